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
// issues the MMAs, warps 4-7 and 8-11 are the epilogues of the accumulator's
// two halves of 128 columns. Three modes:
//   kPair    two CTAs (cta_group::2) share a tile of 256 tokens: each loads its
//            128 tokens and half of the weight rows, so a block costs a CTA 32
//            KB of L2 reads instead of 48. Many tokens a group.
//   kSingle  one CTA a tile, fewer token rows loaded when groups are small: the
//            weights' stream bounds it.
//   kSplit   few tiles: a cluster of up to 8 CTAs shares a tile's blocks; the
//            partial sums meet in distributed shared memory, added in rank
//            order.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdlib>
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

// A whole warp's wait, first without the suspending form (a barrier that is
// ready already costs the least so). One that ran out is recorded where the
// caller gave a word for it, and every later one is skipped.
struct Waiter {
    uint32_t *err;
    bool failed = false;
    __device__ void operator()(uint64_t *bar, uint32_t parity) {
        const uint32_t a = smem_u32(bar);
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(done)
            : "r"(a), "r"(parity)
            : "memory");
        if (__all_sync(0xffffffffu, done) || failed) return;
        for (int i = 0; i < kPoll; ++i) {
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
// An arrival on this CTA's barrier (PAIR: on the leader's)
template <bool PAIR>
__device__ __forceinline__ void arrive(uint64_t *bar) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .b32 r;\n\t"
            "mapa.shared::cluster.u32 r, %0, 0;\n\t"
            "mbarrier.arrive.shared::cluster.b64 _, [r];\n\t}\n" ::"r"(smem_u32(bar))
            : "memory");
    else
        mbar_arrive(bar);
}
template <bool PAIR>
__device__ __forceinline__ bool rank_issues(int rank) {
    return !PAIR || rank == 0;
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
__device__ __forceinline__ uint32_t map_cluster(uint32_t saddr, int cta) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(saddr), "r"(cta));
    return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// ------------------------------------------------------- groups and tiles

struct Groups {
    int pre[kMaxGroups + 1];     // token tiles before group e
    int beg[kMaxGroups], end[kMaxGroups];
};

// Warp 0 fills the groups' rows, clamped to [0, P] and to ascending order
// whatever the offsets hold, and the running count of their token tiles.
__device__ __forceinline__ void build_groups(const GmmArgs &a, Groups &g, int rows_per_tile) {
    const int lane = threadIdx.x & 31;
    const int per = (a.E + 31) / 32, e0 = lane * per;
    int sum = 0;
    for (int e = e0; e < min(e0 + per, a.E); ++e) {
        const int b = min(max(__ldg(a.off + e), 0), a.P), n = min(max(__ldg(a.off + e + 1), b), a.P);
        g.beg[e] = b;
        g.end[e] = n;
        sum += (n - b + rows_per_tile - 1) / rows_per_tile;
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    int at = inc - sum;
    for (int e = e0; e < min(e0 + per, a.E); ++e) {
        g.pre[e] = at;
        at += (g.end[e] - g.beg[e] + rows_per_tile - 1) / rows_per_tile;
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

enum Mode { kSingle = 0, kSplit = 1, kPair = 2 };

constexpr int kAccCols = 256;                  // accumulator columns: two halves of 128
constexpr int kThreads = 384;                  // TMA, MMA, two idle warps, eight epilogue warps
constexpr int kCtlRegs = 40, kEpiRegs = 232;   // setmaxnreg: 128 x 40 + 256 x 232 = 384 x 168
constexpr int kGroup = 4, kSlots = 3;          // scale blocks of a slot of staged scales, and the slots
constexpr int kMaxStages = 8;
constexpr int kRingBytes = 160 * 1024;
constexpr int kPartPitch = 257;                // floats of a row of partial sums (kSplit)
constexpr int kPatch = 4096;                   // an epilogue warp's output staging: 32 rows of 128 bytes
constexpr size_t kSmem = 1024 + kRingBytes + 8 * kPatch;

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
    int box;             // weight rows of one TMA copy (256, 128 or 64)
    int stages;
    int split;           // kSplit: CTAs of a cluster
    int weights_first;   // the first stages' weights may be read before the kernel's predecessor has finished
};

// The 32 rows a warp's lanes hold, through its patch of shared memory, so that
// a store instruction writes whole rows: lane `lane` puts CH 16-byte chunks of
// its row (put), and CH lanes then write each row (flush). A thread storing its
// own row, 16 bytes in each of 32 rows an instruction, took 12800 cycles of a
// 128 x 256 tile; this takes 1400.
template <int CH>
struct RowStore {
    uint8_t *patch;
    int lane;
    __device__ static int at(int row, int c) {
        return row * (CH * 16) + 16 * (c ^ (CH == 8 ? row & 7 : (row >> 1) & 3));
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
    __shared__ uint32_t s_amax[GLU ? 2 * kLanes : 1];
    // staged products of token and weight scales: [slot][block][half, or gate / up][row]
    __shared__ float s_scale[FP8 ? kSlots * kGroup * 2 * kLanes : 1];
    __shared__ uint64_t sc_full[kSlots], sc_empty[kSlots];
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
            mbar_init(&acc_empty[i], PAIR ? 16 : 8);
        }
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&sc_full[i], 2);
            mbar_init(&sc_empty[i], 8);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
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
        } else if (warp == 1 && rank_issues<PAIR>(rank)) {
            // ---- MMA issuer: the sum of one scale block (e4m3) or of a tile
            // (bf16) at a time
            constexpr uint32_t idesc = idesc_of(FP8, PAIR ? 256 : 128, kAccCols);
            int s = 0;
            uint32_t phase = 0, u = 0, uphase = 1;
            for (int tile = first; tile < tiles; tile += step) {
                for (int kb = kb0; kb < kb1; ++kb) {
                    const bool fresh = FP8 || kb == kb0, last = FP8 || kb == kb1 - 1;
                    wait(&full[s], phase);
                    if (fresh) wait(&acc_empty[u], uphase);
                    tc_fence_after();
                    const uint32_t st = sbase + s * stage_bytes, d = tmem + u * kAccCols;
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
        else if (FP8 && warp >= 2) {
            // ---- scales: warps 2 and 3 stage the products of the scales for
            // the epilogue, a few blocks ahead of it. (Loaded by the epilogue
            // itself, however far ahead, they cost it their latency in every
            // block: 1240 cycles a block against 640.)
            const int l = tid - 64;                 // rows l and l + 64
            const int NB = (a.N + kScaleBlock - 1) / kScaleBlock, units = kb1 - kb0;
            int slot = 0;
            uint32_t phase = 1;
            for (int tile = first; tile < tiles; tile += step) {
                const Tile t = locate(a, s_g, tile, ntiles, tile_rows);
                const int nb = GLU ? t.nt : 2 * t.nt;
                const float *w0 = a.sw0 + ((size_t)t.e * NB + nb) * a.KB + kb0;
                const float *w1 = GLU ? a.sw1 + ((size_t)t.e * NB + nb) * a.KB + kb0 : w0 + (nb + 1 < NB ? a.KB : 0);
                const int r = t.row0 + (PAIR ? kLanes * rank : 0) + l;
                const float *x0 = a.sx + (size_t)kb0 * a.P + min(r, a.P - 1), *x1 = x0 + min(64, a.P - 1 - min(r, a.P - 1));
                for (int i0 = 0; i0 < units; i0 += kGroup) {
                    float v[kGroup][4];
#pragma unroll
                    for (int z = 0; z < kGroup; ++z) {
                        const int i = min(i0 + z, units - 1);
                        v[z][0] = __ldg(x0 + (size_t)i * a.P);
                        v[z][1] = __ldg(x1 + (size_t)i * a.P);
                        v[z][2] = __ldg(w0 + i);
                        v[z][3] = __ldg(w1 + i);
                    }
                    wait(&sc_empty[slot], phase);
                    float *to = s_scale + slot * kGroup * 2 * kLanes + l;
#pragma unroll
                    for (int z = 0; z < kGroup; ++z, to += 2 * kLanes) {
                        to[0] = v[z][0] * v[z][2];
                        to[64] = v[z][1] * v[z][2];
                        to[kLanes] = v[z][0] * v[z][3];
                        to[kLanes + 64] = v[z][1] * v[z][3];
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
        // ---- epilogue: thread = one token, one half of the tile's columns:
        // 128 weight rows, or (gate/up) 64 of each matrix
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kEpiRegs));
        const int q = warp & 3, half = (warp - 4) >> 2, row = 32 * q + lane;
        const bool busy = 32 * q < bm;              // lanes that hold token rows at all
        uint8_t *const patch = smem_raw + (sbase - smem_u32(smem_raw)) + kRingBytes + (warp - 4) * kPatch;
        const uint32_t tq = tmem + ((uint32_t)(32 * q) << 16) + half * 128;
        uint32_t un = 0, sphase = 0;
        int slot = 0;
        for (int tile = first; tile < tiles; tile += step) {
            const Tile t = locate(a, s_g, tile, ntiles, tile_rows);
            const int r = t.row0 + (PAIR ? kLanes * rank : 0) + row;
            const bool live = row < bm && r < t.end;
            const int n0 = t.nt * kOutCols + half * (kOutCols / 2);   // its first output column
            uint64_t acc[64];                       // 128 float32 sums
            if (FP8) {
#pragma unroll
                for (int j = 0; j < 64; ++j) acc[j] = 0;
            }
            const int units = FP8 ? kb1 - kb0 : 1;
            for (int i0 = 0; i0 < units; i0 += kGroup) {
                if (FP8) wait(&sc_full[slot], sphase);
                const float *sc = s_scale + slot * kGroup * 2 * kLanes + row;
#pragma unroll
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
                    wait(&acc_full[u], (un >> 1) & 1);
                    ++un;
                    tc_fence_after();
                    uint32_t dv[2][32];
                    auto add = [&](int c) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const uint64_t v = pack2(dv[c & 1][2 * j], dv[c & 1][2 * j + 1]);
                            if (FP8) fma2(acc[16 * c + j], v, c < 2 ? s0 : s1);
                            else acc[16 * c + j] = v;
                        }
                    };
                    if (busy) {
                        tmem_ld32(td, dv[0]);
                        tmem_ld32(td + 32, dv[1]);
                        tmem_wait_ld();
                        add(0);
                        tmem_ld32(td + 64, dv[0]);
                        add(1);
                        tmem_ld32(td + 96, dv[1]);
                        tmem_wait_ld();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive<PAIR>(&acc_empty[u]);
                    if (busy) {
                        add(2);
                        add(3);
                    }
                }
                if (FP8) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sc_empty[slot]);
                    if (++slot == kSlots) {
                        slot = 0;
                        sphase ^= 1;
                    }
                }
            }
            if (SPLIT) {
                // the ring is idle: this CTA's sums, [row][column], rows at
                // a pitch of 257 so that lanes (rows) meet no bank twice and
                // the others read a row's columns in whole lines
                float *part = reinterpret_cast<float *>(smem_raw + (sbase - smem_u32(smem_raw)));
                if (row < bm) {
                    float *to = part + row * kPartPitch + half * 128;
#pragma unroll
                    for (int j = 0; j < 64; ++j) {
                        to[2 * j] = lo2(acc[j]);
                        to[2 * j + 1] = hi2(acc[j]);
                    }
                }
            } else if (GLU) {
                // 64 activations of the token's group of 128; the largest of
                // all 128 with the other half's warp
                uint32_t m = 0, v[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    v[j] = glu_pair(lo2(acc[j]), hi2(acc[j]), lo2(acc[32 + j]), hi2(acc[32 + j]), a.act);
                    if (n0 + 2 * j < a.N) m = __vmaxu2(m, v[j] & 0x7FFF7FFFu);
                }
                m = max(m & 0xFFFFu, m >> 16);
                s_amax[half * kLanes + row] = m;
                bar_sync(1, 256);
                m = max(m, s_amax[(half ^ 1) * kLanes + row]);
                bar_sync(1, 256);                   // read before the next tile's
                const QScale qs = qscale(m);
                const RowStore<4> rows{patch, lane};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[4];
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const uint32_t x0 = v[8 * c + 2 * z], x1 = v[8 * c + 2 * z + 1];
                        w[z] = cvt_e4m3x2(quotient(bf_lo(x0), qs), quotient(bf_hi(x0), qs)) |
                               (cvt_e4m3x2(quotient(bf_lo(x1), qs), quotient(bf_hi(x1), qs)) << 16);
                    }
                    rows.put(c, w[0], w[1], w[2], w[3]);
                }
                rows.flush(a.q_out + n0, a.N, live ? r : -1, a.N - n0);
                if (half == 0 && live) a.s_out[(size_t)t.nt * a.P + r] = qs.s;
            } else {
                const int o = live ? (a.map ? a.map[r] : r) : -1;
                const RowStore<8> rows{patch, lane};
                if (a.out_f32) {
                    uint8_t *y = reinterpret_cast<uint8_t *>(static_cast<float *>(a.out) + n0);
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const uint64_t x0 = acc[16 * h + 2 * c], x1 = acc[16 * h + 2 * c + 1];
                            rows.put(c, (uint32_t)x0, (uint32_t)(x0 >> 32), (uint32_t)x1, (uint32_t)(x1 >> 32));
                        }
                        rows.flush(y + 128 * h, 4 * a.out_stride, o, 4 * (a.N - n0) - 128 * h);
                    }
                } else {
                    const float rs = a.row_scale && o >= 0 ? a.row_scale[o] : 1.0f;
                    uint8_t *y = reinterpret_cast<uint8_t *>(static_cast<uint16_t *>(a.out) + n0);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            uint32_t w[4];
#pragma unroll
                            for (int z = 0; z < 4; ++z) {
                                const uint64_t x = acc[32 * h + 4 * c + z];
                                w[z] = cvt_bf16x2(lo2(x), hi2(x));
                                if (a.row_scale) w[z] = cvt_bf16x2(bf_lo(w[z]) * rs, bf_hi(w[z]) * rs);
                            }
                            rows.put(c, w[0], w[1], w[2], w[3]);
                        }
                        rows.flush(y + 128 * h, 2 * a.out_stride, o, 2 * (a.N - n0) - 128 * h);
                    }
                }
            }
        }
        __syncwarp();
        if (SPLIT) {
            // Each CTA adds up and stores its share of the tile: a warp takes 32
            // columns of a row, or (gate/up) a row's 128 activations.
            cluster_arrive_wait();
            if (first < tiles) {
                const Tile t = locate(a, s_g, first, ntiles, tile_rows);
                const int np = min(bm, t.end - t.row0);
                uint32_t peer[8];
    #pragma unroll
                for (int c = 0; c < 8; ++c) peer[c] = map_cluster(sbase, min(c, S - 1));
                // the cluster's sums of N (row, column)s, every load in flight
                // before the first is used
                auto sums = [&](auto &v, const auto &at) {
                    constexpr int N = sizeof(v) / sizeof(float);
                    float x[N][8];
    #pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (c < S)
    #pragma unroll
                            for (int n = 0; n < N; ++n) x[n][c] = ld_cluster(peer[c] + 4 * at(n));
    #pragma unroll
                    for (int n = 0; n < N; ++n) v[n] = 0.0f;
    #pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (c < S)
    #pragma unroll
                            for (int n = 0; n < N; ++n) v[n] += x[n][c];
                };
                if (GLU) {
                    for (int u = (warp - 4) * S + rank; u < np; u += 8 * S) {
                        float g[8], v[4];            // gate and up of this lane's four columns
                        uint32_t m = 0;
                        sums(g, [&](int n) {
                            const int c = lane + 32 * (n & 3);
                            return u * kPartPitch + (c >> 6) * 128 + (c & 63) + 64 * (n >> 2);
                        });
    #pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t y = glu_pair(g[i], 0.0f, g[4 + i], 0.0f, a.act);
                            v[i] = bf_lo(y);
                            if (t.nt * 128 + lane + 32 * i < a.N) m = max(m, y & 0x7FFFu);
                        }
                        const QScale qs = qscale(__reduce_max_sync(0xffffffffu, m));
                        const size_t r = (size_t)(t.row0 + u);
    #pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int n = t.nt * 128 + lane + 32 * i;
                            if (n < a.N) a.q_out[r * a.N + n] = (uint8_t)cvt_e4m3x2(quotient(v[i], qs), 0.0f);
                        }
                        if (lane == 0) a.s_out[(size_t)t.nt * a.P + r] = qs.s;
                    }
                } else {
                    // 32 columns of a row a warp and step, four steps at a time
                    constexpr int kSteps = 4;
                    const int step8 = 8 * S, total = 8 * np;
                    for (int u0 = (warp - 4) * S + rank; u0 < total; u0 += kSteps * step8) {
                        float v[kSteps];
                        sums(v, [&](int n) {
                            const int u = min(u0 + n * step8, total - 1);
                            return (u >> 3) * kPartPitch + (u & 7) * 32 + lane;
                        });
    #pragma unroll
                        for (int k = 0; k < kSteps; ++k) {
                            const int u = u0 + k * step8, n = t.nt * 256 + (u & 7) * 32 + lane;
                            if (u >= total || n >= a.N) continue;
                            const int r = t.row0 + (u >> 3), o = a.map ? a.map[r] : r;
                            if (a.out_f32) {
                                static_cast<float *>(a.out)[o * a.out_stride + n] = v[k];
                            } else {
                                float y = bf16r(v[k]);
                                if (a.row_scale) y = bf16r(y * a.row_scale[o]);
                                static_cast<uint16_t *>(a.out)[o * a.out_stride + n] = f32_to_bf16(y);
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
    if (n * kThreads < 128 * kCtlRegs + 256 * kEpiRegs)
        return set_error(VQMOE_LAUNCH_FAILED, "gmm_kernel: built with %d registers a thread", n);
    return VQMOE_OK;
}

static bool byte_map(CUtensorMap *m, const void *base, size_t rows, size_t row_bytes, size_t pitch, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    return encode_tma_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, dims, pitch, box) == CUDA_SUCCESS;
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
    // groups that can have rows, their mean rows, and (a bound on) the tiles of `rows` token rows
    const int groups = std::min(a.E, a.P), mean = (a.P + groups - 1) / groups;
    const long long ntiles = (a.N + (glu ? 127 : 255)) / (glu ? 128 : 256);
    auto tiles_of = [&](int rows) {
        return ntiles * (a.off ? std::min<long long>(a.P, a.P / rows + groups) : (a.P + rows - 1) / rows);
    };
    Plan p{};
    p.bm = mean <= 24 ? 32 : mean <= 48 ? 64 : 128;
    p.split = 1;
    const char *env = getenv("GMM_MODE");
    int mode = mean > 128 ? kPair : kSingle;
    if (env) mode = atoi(env);
    if (const char *b = getenv("GMM_BM")) p.bm = atoi(b);
    if (mode != kPair) {
        while (p.split < 8 && tiles_of(p.bm) * p.split * 2 <= sms && p.split * 4 <= a.KB) p.split *= 2;
        mode = p.split > 1 ? kSplit : kSingle;
    } else {
        p.bm = kLanes;
    }
    const int stage = p.bm * 128 + (mode == kPair ? 128 : 256) * 128;
    p.stages = std::min(kMaxStages, kRingBytes / stage);
    p.box = glu ? 64 : mode == kPair ? 128 : 256;
    p.weights_first = pdl_weights && !a.off && mode != kPair;
    const int cluster = mode == kPair ? 2 : p.split;
    const long long tiles = std::min<long long>(tiles_of(mode == kPair ? 256 : p.bm), 1 << 20);
    const int grid = mode == kSplit ? (int)tiles * p.split
                     : mode == kPair ? 2 * (int)std::min<long long>(tiles, sms / 2)
                                     : (int)std::min<long long>(tiles, sms);
    CUtensorMap mx, m0, m1;
    const size_t wrows = (size_t)a.E * a.N;
    if (!byte_map(&mx, x, a.P, row_bytes, x_pitch, p.bm) || !byte_map(&m0, w0, wrows, row_bytes, row_bytes, p.box) ||
        !byte_map(&m1, glu ? w1 : w0, wrows, row_bytes, row_bytes, p.box))
        return set_error(VQMOE_LAUNCH_FAILED, "grouped product: tensor map");
    const void *fn = mode == kPair    ? kernel_of<kPair>(glu, fp8)
                     : mode == kSplit ? kernel_of<kSplit>(glu, fp8)
                                      : kernel_of<kSingle>(glu, fp8);
    vqmoe_status s = check_registers(fn);
    if (s != VQMOE_OK || (s = ensure_dynamic_smem(fn, kSmem, "gmm_kernel")) != VQMOE_OK) return s;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
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

// A half warp per group of 128: 8 values a lane, the largest |bf16| by
// integer comparison of the bits (a NaN compares above an infinity, and both
// above every finite value).
template <bool ORDER>
__global__ void __launch_bounds__(256)
    quantize_kernel(const uint16_t *__restrict__ x, long long rows, int cols, long long x_stride,
                    uint8_t *__restrict__ q, float *__restrict__ s, long long s_row, long long s_group,
                    const QuantOrder o) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 15;
    const int groups = (cols + kScaleBlock - 1) / kScaleBlock;
    const long long total = rows * groups, half = (long long)gridDim.x * 16;
    // every lane of a warp runs the same trips (the shuffles need both halves)
    const long long h0 = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const long long trips = (total + half - 1) / half;
    for (long long i = 0; i < trips; ++i) {
        const long long g = h0 + i * half;
        const bool in = g < total;
        const long long row = in ? g / groups : 0;
        const int grp = in ? (int)(g - row * groups) : 0;
        const int c = grp * kScaleBlock + lane * 8;
        const bool live = in && c < cols;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live) v = __ldg(reinterpret_cast<const uint4 *>(x + row * x_stride + c));
        uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu),
                              __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
        const QScale qs = qscale(max(m & 0xFFFFu, m >> 16));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t b[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) b[z] = cvt_e4m3x2(quotient(bf_lo(w[z]), qs), quotient(bf_hi(w[z]), qs));
        const uint2 r = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
        if (!ORDER) {
            if (live) *reinterpret_cast<uint2 *>(q + row * cols + c) = r;
            if (in && lane == 0) s[row * s_row + grp * s_group] = qs.s;
        } else if (in) {
            const int k = o.per_pair ? 1 : o.k;
            for (int z = 0; z < k; ++z) {
                const long long p = row * k + z;
                const int rk = __ldg(o.rank + p);
                if (rk < 0) continue;               // no such expert: the pair has no place
                const long long at = __ldg(o.off + __ldg(o.inds + p)) + rk;
                if (live) *reinterpret_cast<uint2 *>(q + at * cols + c) = r;
                if (lane == 0) s[at * s_row + grp * s_group] = qs.s;
            }
        }
    }
}

}  // namespace gm

vqmoe_status launch_quantize_fp8(const void *x, long long rows, int cols, long long x_stride, uint8_t *q, float *s,
                                 long long s_row, long long s_group, const QuantOrder *order, cudaStream_t stream) {
    if (rows <= 0) return VQMOE_OK;
    const long long groups = rows * ((cols + kScaleBlock - 1) / kScaleBlock);
    const int grid = (int)std::min<long long>((groups + 15) / 16, (long long)sm_count() * 16);
    const uint16_t *xp = static_cast<const uint16_t *>(x);
    if (order)
        gm::quantize_kernel<true><<<grid, 256, 0, stream>>>(xp, rows, cols, x_stride, q, s, s_row, s_group, *order);
    else
        gm::quantize_kernel<false><<<grid, 256, 0, stream>>>(xp, rows, cols, x_stride, q, s, s_row, s_group, QuantOrder{});
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
