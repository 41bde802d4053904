// Products of token rows with their group's weights, y[r] = x[r] W[e(r)]^T,
// on the 5th-generation tensor cores: bf16 operands, or e4m3 operands with a
// float32 scale for each token and 128 inputs (sx) and for each 128 x 128
// weights (sw):
//   y[r][n] = sum_b sx[b][r] sw[e][n / 128][b] (sum over block b of x w)
// A block's inner sum is four tcgen05.mma of 32 inputs into TMEM; the scales
// differ from block to block, so the epilogue warps read every block's sum
// back and add it, scaled, to float32 registers, while the tensor core works
// on the next blocks (TMEM holds two to four of them). bf16 needs none of
// this: a tile's whole sum stays in TMEM.
//
// The groups' rows are contiguous (`off`, on the device): a tile is rows of
// one group. Rows past the group's end that a TMA box brings along belong to
// another group or are zero; they are lines of the product that are never
// stored.
//
// Two kernels, by which operand takes the 128 lanes of the accumulator:
//   tok_n_kernel  weight rows on the lanes, 16-128 tokens as the MMA's N:
//                 few tokens a group. Bound by streaming the weights; with
//                 few tiles a cluster of CTAs shares a tile's inputs and adds
//                 its partial sums through distributed shared memory.
//   tok_m_kernel  128 tokens on the lanes, 256 weight rows as N: many tokens a
//                 group. Bound by the tensor cores and by feeding them.
// Both run persistent CTAs of specialised warps: one issues TMA copies into a
// ring of 128-byte-swizzled stages, one issues the MMAs, the others are the
// epilogue.
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
constexpr int kTileBytes = kLanes * 128;       // 128 rows x 128 bytes
constexpr int kChunk = 16;                     // scale blocks staged at a time (tok_n)

// A wait that ran out is recorded where the caller gave a word for it.
struct Waiter {
    uint32_t *err;
    bool failed = false;
    __device__ void operator()(uint64_t *bar, uint32_t parity) {
        if (failed) return;
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
            if (done) return;
        }
        failed = true;
        if (err) atomicExch(err, kWaitPipeline);
    }
};

template <bool FP8>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
    if (FP8)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
            "l"(ad), "l"(bd), "r"(idesc), "r"(accumulate)
            : "memory");
}

// D f32, A and B e4m3 (kind::f8f6f4) or bf16 (kind::f16), both K-major
constexpr uint32_t idesc_of(bool fp8, int n) {
    return (1u << 4) | (fp8 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kLanes >> 4) << 24);
}

// d += s * v, two float32 at a time
__device__ __forceinline__ void fma2(float &d0, float &d1, uint32_t v0, uint32_t v1, float s0, float s1) {
    asm("{\n\t.reg .b64 a, b, c;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "mov.b64 c, {%0, %1};\n\t"
        "fma.rn.f32x2 c, a, b, c;\n\t"
        "mov.b64 {%0, %1}, c;\n\t}\n"
        : "+f"(d0), "+f"(d1)
        : "f"(__uint_as_float(v0)), "f"(__uint_as_float(v1)), "f"(s0), "f"(s1));
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t *v) {
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
__device__ __forceinline__ float ld_cluster(uint32_t saddr, uint32_t cta) {
    uint32_t r;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(saddr), "r"(cta));
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(r) : "memory");
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

// bf16(bf16(act(g)) * u), g and u the bf16 outputs of the gate and up products
__device__ __forceinline__ float glu_value(float g, float u, int act) {
    const float gb = bf16r(g);
    return bf16r(bf16r(act == VQMOE_ACT_GEGLU ? gelu_tanh_f32(gb) : silu_f32(gb)) * bf16r(u));
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

// ------------------------------------------- few tokens: tokens as the MMA's N

template <int BN, int NMAT, bool FP8, bool SPLIT>
struct NCfg {
    static constexpr int kStageBytes = NMAT * kTileBytes + BN * 128;
    static constexpr int kBudget = 196 * 1024;                     // one CTA an SM
    static constexpr int kPartBytes = SPLIT ? NMAT * BN * kLanes * 4 : 0;
    static constexpr int kOutBytes = BN * kLanes * 2;
    static constexpr int kFit = (kBudget - kPartBytes - kOutBytes) / kStageBytes;
    static constexpr int kStages = kFit > 12 ? 12 : kFit;
    static constexpr int kCols = NMAT * BN;                        // one accumulator
    static constexpr int kUnits = 512 / kCols > 4 ? 4 : 512 / kCols;
    static constexpr int kWant = kUnits * kCols;
    static constexpr int kAlloc = kWant <= 32 ? 32 : kWant <= 64 ? 64 : kWant <= 128 ? 128 : kWant <= 256 ? 256 : 512;
    static constexpr size_t kSmem = 1024 + (size_t)kStages * kStageBytes + kPartBytes + kOutBytes;
    static_assert(kStages >= 2 && kUnits >= 1, "tile too large");
};

constexpr int kNThreads = 192;

template <int BN, int NMAT, bool FP8, bool SPLIT>
__global__ void __launch_bounds__(kNThreads)
    tok_n_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw0,
                 const __grid_constant__ CUtensorMap tw1, const GmmArgs a, int weights_first) {
    using C = NCfg<BN, NMAT, FP8, SPLIT>;
    constexpr bool GLU = NMAT == 2;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[C::kStages], empty[C::kStages], acc_full[C::kUnits], acc_empty[C::kUnits];
    __shared__ uint32_t s_tmem;
    __shared__ Groups s_g;
    __shared__ __align__(16) float s_sx[FP8 ? kChunk * BN : 1];
    __shared__ float s_rs[BN];
    __shared__ int s_row[BN];
    __shared__ uint32_t s_amax[GLU ? BN : 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *const sgen = smem_raw + (sbase - smem_u32(smem_raw));
    float *const s_part = reinterpret_cast<float *>(sgen + C::kStages * C::kStageBytes);
    uint16_t *const s_out = reinterpret_cast<uint16_t *>(sgen + C::kStages * C::kStageBytes + C::kPartBytes);
    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < C::kUnits; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)),
                     "r"(C::kAlloc)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    const int ntiles = (a.N + kLanes - 1) / kLanes;
    const int S = SPLIT ? a.split : 1, part = SPLIT ? blockIdx.x % S : 0;
    const int first = blockIdx.x / S, step = gridDim.x / S;
    const int kb0 = (int)((long long)a.KB * part / S), kb1 = (int)((long long)a.KB * (part + 1) / S);
    Waiter wait{a.err};
    // A dense product's weights do not depend on the kernel before this one:
    // the first stages' weights are on their way before its result is waited
    // for.
    int early = 0;
    if (weights_first && warp == 0) {
        const int dense_tiles = ((a.P + BN - 1) / BN) * ntiles;
        if (first < dense_tiles) early = min(C::kStages, kb1 - kb0);
        if (elect_one()) {
            const int n0 = (first % ntiles) * kLanes;
            for (int s = 0; s < early; ++s) {
                const uint32_t st = sbase + s * C::kStageBytes;
                arrive_expect_tx(&full[s], C::kStageBytes);
                tma_load_2d(st, &tw0, (kb0 + s) * 128, n0, &full[s]);
                if (GLU) tma_load_2d(st + kTileBytes, &tw1, (kb0 + s) * 128, n0, &full[s]);
            }
        }
        __syncwarp();
    }
    pdl_wait();
    pdl_trigger();
    if (a.off && warp == 0) build_groups(a, s_g, BN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const int tiles = (a.off ? s_g.pre[a.E] : (a.P + BN - 1) / BN) * ntiles;
    if (warp == 0) {
        // ---- TMA producer
        int s = 0;
        uint32_t phase = 1;                         // an empty stage's first wait passes
        for (int tile = first; tile < tiles; tile += step) {
            const Tile t = locate(a, s_g, tile, ntiles, BN);
            const int wrow = t.e * a.N + t.nt * kLanes;
            for (int kb = kb0; kb < kb1; ++kb) {
                const uint32_t st = sbase + s * C::kStageBytes;
                wait(&empty[s], phase);
                if (elect_one()) {
                    if (early <= 0) {
                        arrive_expect_tx(&full[s], C::kStageBytes);
                        tma_load_2d(st, &tw0, kb * 128, wrow, &full[s]);
                        if (GLU) tma_load_2d(st + kTileBytes, &tw1, kb * 128, wrow, &full[s]);
                    }
                    tma_load_2d(st + NMAT * kTileBytes, &tx, kb * 128, t.row0, &full[s]);
                }
                __syncwarp();
                --early;
                if (++s == C::kStages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        // ---- MMA issuer: one accumulator a scale block (e4m3) or a tile (bf16)
        constexpr uint32_t idesc = idesc_of(FP8, BN);
        int s = 0, u = 0;
        uint32_t phase = 0, uphase = 1;
        for (int tile = first; tile < tiles; tile += step) {
            for (int kb = kb0; kb < kb1; ++kb) {
                const bool fresh = FP8 || kb == kb0, last = FP8 || kb == kb1 - 1;
                if (fresh) wait(&acc_empty[u], uphase);
                wait(&full[s], phase);
                tc_fence_after();
                const uint32_t st = sbase + s * C::kStageBytes, d = tmem + u * C::kCols;
                if (elect_one()) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int m = 0; m < NMAT; ++m)
                            mma_ss<FP8>(d + m * BN, sw128_desc(st + m * kTileBytes + 32 * q),
                                        sw128_desc(st + NMAT * kTileBytes + 32 * q), idesc, !fresh || q > 0);
                    tc_commit(&empty[s]);
                    if (last) tc_commit(&acc_full[u]);
                }
                __syncwarp();
                if (++s == C::kStages) {
                    s = 0;
                    phase ^= 1;
                }
                if (last && ++u == C::kUnits) {
                    u = 0;
                    uphase ^= 1;
                }
            }
        }
    } else {
        // ---- epilogue: thread = one weight row, warp w the TMEM lanes 32 (w % 4) ..
        const int q = warp & 3, row = 32 * q + lane, et = tid - 64;
        uint32_t un = 0;
        for (int tile = first; tile < tiles; tile += step) {
            const Tile t = locate(a, s_g, tile, ntiles, BN);
            const int np = min(BN, t.end - t.row0);
            float acc[NMAT][BN];
#pragma unroll
            for (int m = 0; m < NMAT; ++m)
#pragma unroll
                for (int j = 0; j < BN; ++j) acc[m][j] = 0.0f;
            bar_sync(1, 128);                       // the last tile's staging has been read
            for (int j = et; j < BN; j += 128) {
                const int r = t.row0 + j;
                const int o = j < np ? (a.map ? a.map[r] : r) : -1;
                s_row[j] = o;
                s_rs[j] = a.row_scale && o >= 0 ? a.row_scale[o] : 1.0f;
                if (GLU) s_amax[j] = 0;
            }
            const float *w0 = nullptr, *w1 = nullptr;
            if (FP8) {
                const size_t at = ((size_t)t.e * ntiles + t.nt) * a.KB;
                w0 = a.sw0 + at;
                w1 = GLU ? a.sw1 + at : nullptr;
            }
            const uint32_t tq = tmem + ((uint32_t)(32 * q) << 16);
            const int units = FP8 ? kb1 - kb0 : 1;
            for (int i = 0; i < units; ++i, ++un) {
                if (FP8 && i % kChunk == 0) {
                    // the next blocks' token scales
                    if (i) bar_sync(1, 128);
                    const int nb = min(kChunk, units - i);
                    for (int v = et; v < nb * BN; v += 128) {
                        const int b = v / BN, j = v % BN;
                        s_sx[v] = j < np ? a.sx[(size_t)(kb0 + i + b) * a.P + t.row0 + j] : 0.0f;
                    }
                    bar_sync(1, 128);
                }
                const float f0 = FP8 ? __ldg(w0 + kb0 + i) : 1.0f, f1 = FP8 && GLU ? __ldg(w1 + kb0 + i) : 1.0f;
                const uint32_t u = un % C::kUnits;
                wait(&acc_full[u], (un / C::kUnits) & 1);
                tc_fence_after();
                constexpr int kStep = BN < 32 ? 16 : 32;
#pragma unroll
                for (int c = 0; c < BN / kStep; ++c) {
                    uint32_t dv[NMAT][32];
#pragma unroll
                    for (int m = 0; m < NMAT; ++m) {
                        if constexpr (kStep == 16) tmem_ld16(tq + u * C::kCols + m * BN + c * 16, dv[m]);
                        else tmem_ld32(tq + u * C::kCols + m * BN + c * 32, dv[m]);
                    }
                    tmem_wait_ld();
                    if (c == BN / kStep - 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&acc_empty[u]);
                    }
                    if (FP8) {
                        const float4 *sx = reinterpret_cast<const float4 *>(s_sx + (i % kChunk) * BN + c * kStep);
#pragma unroll
                        for (int j4 = 0; j4 < kStep / 4; ++j4) {
                            const float4 s = sx[j4];
                            const int j = c * kStep + 4 * j4;
                            fma2(acc[0][j], acc[0][j + 1], dv[0][4 * j4], dv[0][4 * j4 + 1], s.x * f0, s.y * f0);
                            fma2(acc[0][j + 2], acc[0][j + 3], dv[0][4 * j4 + 2], dv[0][4 * j4 + 3], s.z * f0,
                                 s.w * f0);
                            if (GLU) {
                                constexpr int M = NMAT - 1;
                                fma2(acc[M][j], acc[M][j + 1], dv[M][4 * j4], dv[M][4 * j4 + 1], s.x * f1, s.y * f1);
                                fma2(acc[M][j + 2], acc[M][j + 3], dv[M][4 * j4 + 2], dv[M][4 * j4 + 3], s.z * f1,
                                     s.w * f1);
                            }
                        }
                    } else {
#pragma unroll
                        for (int m = 0; m < NMAT; ++m)
#pragma unroll
                            for (int j = 0; j < kStep; ++j) acc[m][c * kStep + j] = __uint_as_float(dv[m][j]);
                    }
                }
            }
            if (SPLIT) {
#pragma unroll
                for (int m = 0; m < NMAT; ++m)
#pragma unroll
                    for (int j = 0; j < BN; ++j) s_part[(m * BN + j) * kLanes + row] = acc[m][j];
            } else {
                if (!FP8) bar_sync(1, 128);         // s_row, s_rs
#pragma unroll
                for (int j = 0; j < BN; ++j) {
                    float v;
                    if (GLU) {
                        v = glu_value(acc[0][j], acc[NMAT - 1][j], a.act);
                    } else {
                        v = acc[0][j];
                        if (a.out_f32) {
                            const int o = s_row[j], n = t.nt * kLanes + row;
                            if (o >= 0 && n < a.N) static_cast<float *>(a.out)[o * a.out_stride + n] = v;
                            continue;
                        }
                        v = bf16r(v);
                        if (a.row_scale) v = bf16r(v * s_rs[j]);
                    }
                    const uint32_t b = __float_as_uint(v) >> 16;
                    if (GLU) {
                        const uint32_t m = __reduce_max_sync(0xffffffffu,
                                                             t.nt * kLanes + row < a.N ? b & 0x7FFFu : 0u);
                        if (lane == 0) atomicMax(&s_amax[j], m);
                    }
                    s_out[j * kLanes + row] = (uint16_t)b;
                }
            }
            if (!SPLIT) {
                bar_sync(1, 128);
                const int nc = (min(kLanes, a.N - t.nt * kLanes) + 15) / 16;   // 16-column pieces
                for (int v = et; v < np * 8; v += 128) {
                    const int j = v >> 3, c = v & 7;
                    if (c >= nc) continue;
                    const uint4 *p = reinterpret_cast<const uint4 *>(s_out + j * kLanes + c * 16);
                    const uint4 lo = p[0], hi = p[1];
                    if (GLU) {
                        const QScale qs = qscale(s_amax[j]);
                        const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                        uint32_t o[4];
#pragma unroll
                        for (int z = 0; z < 4; ++z)
                            o[z] = cvt_e4m3x2(quotient(bf_lo(w[2 * z]), qs), quotient(bf_hi(w[2 * z]), qs)) |
                                   (cvt_e4m3x2(quotient(bf_lo(w[2 * z + 1]), qs),
                                               quotient(bf_hi(w[2 * z + 1]), qs)) << 16);
                        const size_t r = (size_t)(t.row0 + j);
                        *reinterpret_cast<uint4 *>(a.q_out + r * a.N + t.nt * kLanes + c * 16) =
                            make_uint4(o[0], o[1], o[2], o[3]);
                        if (c == 0) a.s_out[(size_t)t.nt * a.P + r] = qs.s;
                    } else if (!a.out_f32) {
                        uint4 *o = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) +
                                                             s_row[j] * a.out_stride + t.nt * kLanes + c * 16);
                        o[0] = lo;
                        o[1] = hi;
                    }
                }
            }
        }
    }
    __syncwarp();
    if (SPLIT) {
        // the cluster's partial sums, added in rank order: CTA `part` takes
        // its share of the tile's tokens
        cluster_arrive_wait();
        if (warp >= 2 && first < tiles) {
            const Tile t = locate(a, s_g, first, ntiles, BN);
            const int np = min(BN, t.end - t.row0);
            const int row = 32 * (warp & 3) + lane, n = t.nt * kLanes + row;
            const int j0 = BN * part / S, j1 = min(BN * (part + 1) / S, np);
            const uint32_t pbase = smem_u32(s_part);
            for (int j = j0; j < j1; ++j) {
                float v[NMAT];
#pragma unroll
                for (int m = 0; m < NMAT; ++m) {
                    v[m] = 0.0f;
                    for (int c = 0; c < S; ++c) v[m] += ld_cluster(pbase + 4 * ((m * BN + j) * kLanes + row), c);
                }
                if (GLU) {
                    const uint32_t b = __float_as_uint(glu_value(v[0], v[NMAT - 1], a.act)) >> 16;
                    const uint32_t m = __reduce_max_sync(0xffffffffu, n < a.N ? b & 0x7FFFu : 0u);
                    if (lane == 0) atomicMax(&s_amax[j], m);
                    s_out[j * kLanes + row] = (uint16_t)b;
                } else if (n < a.N) {
                    const int o = s_row[j];
                    if (a.out_f32) {
                        static_cast<float *>(a.out)[o * a.out_stride + n] = v[0];
                    } else {
                        float y = bf16r(v[0]);
                        if (a.row_scale) y = bf16r(y * s_rs[j]);
                        static_cast<uint16_t *>(a.out)[o * a.out_stride + n] = f32_to_bf16(y);
                    }
                }
            }
            if (GLU) {
                bar_sync(1, 128);
                for (int j = j0; j < j1; ++j) {
                    const QScale qs = qscale(s_amax[j]);
                    const size_t r = (size_t)(t.row0 + j);
                    if (n < a.N)
                        a.q_out[r * a.N + n] =
                            (uint8_t)cvt_e4m3x2(quotient(bf16_to_f32(s_out[j * kLanes + row]), qs), 0.0f);
                    if (row == 0) a.s_out[(size_t)t.nt * a.P + r] = qs.s;
                }
            }
        }
        __syncwarp();
        cluster_arrive_wait();                      // the others have read this CTA's sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(C::kAlloc) : "memory");
    }
}

// ------------------------------------------ many tokens: tokens as the MMA's M

constexpr int kCols = 256;                     // weight rows of a tile (gate/up: 128 of each)
constexpr int kMStages = 4;
constexpr int kMStageBytes = kTileBytes + kCols * 128;
constexpr size_t kMSmem = 1024 + (size_t)kMStages * kMStageBytes;
constexpr int kMThreads = 384;                 // TMA, MMA, two idle warps, eight epilogue warps
constexpr int kCtlRegs = 40, kEpiRegs = 232;   // setmaxnreg: 128 x 40 + 256 x 232 = 384 x 168

// SwiGLU / GeGLU of two columns, every step rounded to bf16: packed bf16
__device__ __forceinline__ uint32_t glu_pair(float g0, float g1, float u0, float u1, int act) {
    const uint32_t g = cvt_bf16x2(g0, g1), u = cvt_bf16x2(u0, u1);
    const uint32_t a = act == VQMOE_ACT_GEGLU ? cvt_bf16x2(gelu_tanh_f32(bf_lo(g)), gelu_tanh_f32(bf_hi(g)))
                                              : cvt_bf16x2(silu_fast(bf_lo(g)), silu_fast(bf_hi(g)));
    return cvt_bf16x2(bf_lo(a) * bf_lo(u), bf_hi(a) * bf_hi(u));
}

template <bool GLU, bool FP8>
__global__ void __launch_bounds__(kMThreads, 1)
    tok_m_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw0,
                 const __grid_constant__ CUtensorMap tw1, const GmmArgs a) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kMStages], empty[kMStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t s_tmem;
    __shared__ Groups s_g;
    __shared__ uint32_t s_amax[GLU ? 2 * kLanes : 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;
    if (tid == 0) {
        for (int i = 0; i < kMStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], 8);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&s_tmem)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    pdl_wait();
    pdl_trigger();
    if (a.off && warp == 0) build_groups(a, s_g, kLanes);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    constexpr int kOutCols = GLU ? 128 : kCols;    // output columns of a tile
    const int ntiles = (a.N + kOutCols - 1) / kOutCols;
    const int tiles = (a.off ? s_g.pre[a.E] : (a.P + kLanes - 1) / kLanes) * ntiles;
    Waiter wait{a.err};
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kCtlRegs));
        if (warp == 0) {
            // ---- TMA producer
            int s = 0;
            uint32_t phase = 1;
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
                const Tile t = locate(a, s_g, tile, ntiles, kLanes);
                const int wrow = t.e * a.N + t.nt * kOutCols;
                for (int kb = 0; kb < a.KB; ++kb) {
                    const uint32_t st = sbase + s * kMStageBytes;
                    wait(&empty[s], phase);
                    if (elect_one()) {
                        arrive_expect_tx(&full[s], kMStageBytes);
                        tma_load_2d(st, &tx, kb * 128, t.row0, &full[s]);
                        tma_load_2d(st + kTileBytes, &tw0, kb * 128, wrow, &full[s]);
                        if (GLU) tma_load_2d(st + 2 * kTileBytes, &tw1, kb * 128, wrow, &full[s]);
                    }
                    __syncwarp();
                    if (++s == kMStages) {
                        s = 0;
                        phase ^= 1;
                    }
                }
            }
        } else if (warp == 1) {
            // ---- MMA issuer: one accumulator a scale block (e4m3) or a tile (bf16)
            constexpr uint32_t idesc = idesc_of(FP8, kCols);
            int s = 0;
            uint32_t phase = 0, u = 0, uphase = 1;
            for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
                for (int kb = 0; kb < a.KB; ++kb) {
                    const bool fresh = FP8 || kb == 0, last = FP8 || kb == a.KB - 1;
                    if (fresh) wait(&acc_empty[u], uphase);
                    wait(&full[s], phase);
                    tc_fence_after();
                    const uint32_t st = sbase + s * kMStageBytes, d = tmem + u * kCols;
                    if (elect_one()) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            mma_ss<FP8>(d, sw128_desc(st + 32 * q), sw128_desc(st + kTileBytes + 32 * q), idesc,
                                        !fresh || q > 0);
                        tc_commit(&empty[s]);
                        if (last) tc_commit(&acc_full[u]);
                    }
                    __syncwarp();
                    if (++s == kMStages) {
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
    } else {
        // ---- epilogue: thread = one token, half of the tile's columns: 128
        // weight rows, or (gate/up) 64 of each matrix
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kEpiRegs));
        const int q = warp & 3, half = (warp - 4) >> 2, row = 32 * q + lane;
        const uint32_t tq = tmem + ((uint32_t)(32 * q) << 16);
        // its accumulator columns in four pieces of 32
        auto piece = [&](int c) -> uint32_t { return GLU ? 64 * half + (c & 1) * 32 + (c >> 1) * 128 : 128 * half + 32 * c; };
        const int NB = (a.N + kScaleBlock - 1) / kScaleBlock;
        uint32_t un = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            const Tile t = locate(a, s_g, tile, ntiles, kLanes);
            const int r = t.row0 + row;
            const bool live = r < t.end;
            const int n0 = t.nt * kOutCols + piece(0);   // its first output column
            float acc[128];
            const float *w0 = nullptr, *w1 = nullptr;
            if (FP8) {
#pragma unroll
                for (int j = 0; j < 128; ++j) acc[j] = 0.0f;
                const size_t at = ((size_t)t.e * NB + min(n0 / kScaleBlock, NB - 1)) * a.KB;
                w0 = a.sw0 + at;
                w1 = GLU ? a.sw1 + at : w0;
            }
            const int units = FP8 ? a.KB : 1;
            float sx = FP8 && live ? __ldg(a.sx + r) : 0.0f;
            float f0 = FP8 ? __ldg(w0) : 1.0f, f1 = FP8 && GLU ? __ldg(w1) : 1.0f;
            for (int i = 0; i < units; ++i, ++un) {
                const float s0 = sx * f0, s1 = GLU ? sx * f1 : s0;
                if (FP8 && i + 1 < units) {            // the next block's scales
                    if (live) sx = __ldg(a.sx + (size_t)(i + 1) * a.P + r);
                    f0 = __ldg(w0 + i + 1);
                    if (GLU) f1 = __ldg(w1 + i + 1);
                }
                const uint32_t u = un & 1, td = tq + u * kCols;
                wait(&acc_full[u], (un >> 1) & 1);
                tc_fence_after();
                uint32_t dv[2][32];
                auto add = [&](int c) {
                    const float s = c >= 2 ? s1 : s0;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        if (FP8) {
                            fma2(acc[32 * c + j], acc[32 * c + j + 1], dv[c & 1][j], dv[c & 1][j + 1], s, s);
                        } else {
                            acc[32 * c + j] = __uint_as_float(dv[c & 1][j]);
                            acc[32 * c + j + 1] = __uint_as_float(dv[c & 1][j + 1]);
                        }
                    }
                };
                tmem_ld32(td + piece(0), dv[0]);
                tmem_ld32(td + piece(1), dv[1]);
                tmem_wait_ld();
                add(0);
                tmem_ld32(td + piece(2), dv[0]);
                add(1);
                tmem_ld32(td + piece(3), dv[1]);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&acc_empty[u]);
                add(2);
                add(3);
            }
            if (GLU) {
                // 64 activations of the token's group of 128; the largest of
                // all 128 with the other half's warp
                uint32_t m = 0, v[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    v[j] = glu_pair(acc[2 * j], acc[2 * j + 1], acc[64 + 2 * j], acc[65 + 2 * j], a.act);
                    if (n0 + 2 * j < a.N) m = __vmaxu2(m, v[j] & 0x7FFF7FFFu);
                }
                m = max(m & 0xFFFFu, m >> 16);
                s_amax[half * kLanes + row] = m;
                bar_sync(1, 256);
                m = max(m, s_amax[(half ^ 1) * kLanes + row]);
                bar_sync(1, 256);                      // read before the next tile's
                const QScale qs = qscale(m);
                if (live) {
                    uint8_t *o = a.q_out + (size_t)r * a.N + n0;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const uint32_t x0 = v[8 * c + 2 * z], x1 = v[8 * c + 2 * z + 1];
                            w[z] = cvt_e4m3x2(quotient(bf_lo(x0), qs), quotient(bf_hi(x0), qs)) |
                                   (cvt_e4m3x2(quotient(bf_lo(x1), qs), quotient(bf_hi(x1), qs)) << 16);
                        }
                        if (n0 + 16 * c < a.N) reinterpret_cast<uint4 *>(o)[c] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (half == 0) a.s_out[(size_t)t.nt * a.P + r] = qs.s;
                }
            } else if (live) {
                const int o = a.map ? a.map[r] : r;
                if (a.out_f32) {
                    float *p = static_cast<float *>(a.out) + o * a.out_stride + n0;
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (n0 + 4 * c < a.N)
                            reinterpret_cast<float4 *>(p)[c] =
                                make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
                } else {
                    const float rs = a.row_scale ? a.row_scale[o] : 1.0f;
                    uint16_t *p = static_cast<uint16_t *>(a.out) + o * a.out_stride + n0;
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        uint32_t w[4];
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            w[z] = cvt_bf16x2(acc[8 * c + 2 * z], acc[8 * c + 2 * z + 1]);
                            if (a.row_scale) w[z] = cvt_bf16x2(bf_lo(w[z]) * rs, bf_hi(w[z]) * rs);
                        }
                        if (n0 + 8 * c < a.N) reinterpret_cast<uint4 *>(p)[c] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
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
    if (cudaGetDevice(&dev) != cudaSuccess) return check_launch("tok_m_kernel");
    std::lock_guard<std::mutex> lock(mu);
    int &n = regs[{fn, dev}];
    if (!n) {
        cudaFuncAttributes at{};
        if (cudaFuncGetAttributes(&at, fn) != cudaSuccess) return check_launch("tok_m_kernel");
        n = at.numRegs;
    }
    if (n * kMThreads < 128 * kCtlRegs + 256 * kEpiRegs)
        return set_error(VQMOE_LAUNCH_FAILED, "tok_m_kernel: built with %d registers a thread", n);
    return VQMOE_OK;
}

static bool byte_map(CUtensorMap *m, const void *base, size_t rows, size_t row_bytes, size_t pitch, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    return encode_tma_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, dims, pitch, box) == CUDA_SUCCESS;
}

struct Maps {
    CUtensorMap x, w0, w1;
};

static vqmoe_status launch_with(const void *fn, const char *what, Maps &m, const GmmArgs &a, int grid, int threads,
                                size_t smem, int cluster, const int *weights_first, cudaStream_t stream) {
    vqmoe_status s = ensure_dynamic_smem(fn, smem, what);
    if (s != VQMOE_OK) return s;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
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
    int wf = weights_first ? *weights_first : 0;
    void *params[5] = {&m.x, &m.w0, &m.w1, const_cast<GmmArgs *>(&a), &wf};
    if (cudaLaunchKernelExC(&cfg, fn, params) != cudaSuccess) return check_launch(what);
    return VQMOE_OK;
}

template <int BN, int NMAT, bool FP8, bool SPLIT>
static vqmoe_status launch_n(Maps &m, const GmmArgs &a, int tiles, int wf, cudaStream_t stream) {
    using C = NCfg<BN, NMAT, FP8, SPLIT>;
    const int grid = SPLIT ? tiles * a.split : std::min(tiles, sm_count());
    return launch_with(reinterpret_cast<const void *>(&tok_n_kernel<BN, NMAT, FP8, SPLIT>), "tok_n_kernel", m, a, grid,
                       kNThreads, C::kSmem, SPLIT ? a.split : 1, &wf, stream);
}

template <int BN, int NMAT, bool FP8>
static vqmoe_status launch_n2(Maps &m, const GmmArgs &a, int tiles, int wf, cudaStream_t stream) {
    return a.split > 1 ? launch_n<BN, NMAT, FP8, true>(m, a, tiles, wf, stream)
                       : launch_n<BN, NMAT, FP8, false>(m, a, tiles, wf, stream);
}

}  // namespace gm

vqmoe_status launch_gmm(const void *x, size_t x_pitch, const void *w0, const void *w1, size_t row_bytes, bool fp8,
                        GmmArgs a, cudaStream_t stream, bool pdl_weights) {
    using namespace gm;
    const bool glu = w1 != nullptr;
    if (a.P <= 0) return VQMOE_OK;
    if (a.E <= 0 || a.E > kMaxGroups || (!a.off && a.E != 1))
        return set_error(VQMOE_BAD_SHAPE, "grouped product: %d groups (1..%d)", a.E, kMaxGroups);
    if ((long long)a.E * a.N > 0x7FFFFFFFLL - 256 || (long long)a.KB * 128 > 0x7FFFFFFFLL)
        return set_error(VQMOE_BAD_SHAPE, "grouped product: %d groups of %d rows", a.E, a.N);
    // groups that can have rows, and their mean rows
    const int groups = std::min(a.E, a.P), mean = (a.P + groups - 1) / groups;
    const int bn_max = glu ? 64 : 128;
    const char *env = getenv("GMM_M"); const int thr = env ? atoi(env) : bn_max;
    Maps m;
    const size_t wrows = (size_t)a.E * a.N;
    if (mean > thr) {
        if (!byte_map(&m.x, x, a.P, row_bytes, x_pitch, kLanes) ||
            !byte_map(&m.w0, w0, wrows, row_bytes, row_bytes, glu ? 128 : kCols) ||
            !byte_map(&m.w1, glu ? w1 : w0, wrows, row_bytes, row_bytes, 128))
            return set_error(VQMOE_LAUNCH_FAILED, "grouped product: tensor map");
        const int out_cols = glu ? 128 : kCols;
        const long long tiles = ((long long)a.P / kLanes + groups) * ((a.N + out_cols - 1) / out_cols);
        const int grid = (int)std::min<long long>(tiles, sm_count());
        a.split = 1;
        const void *fn = glu   ? reinterpret_cast<const void *>(&tok_m_kernel<true, true>)
                         : fp8 ? reinterpret_cast<const void *>(&tok_m_kernel<false, true>)
                               : reinterpret_cast<const void *>(&tok_m_kernel<false, false>);
        const vqmoe_status s = check_registers(fn);
        if (s != VQMOE_OK) return s;
        return launch_with(fn, "tok_m_kernel", m, a, grid, kMThreads, kMSmem, 1, nullptr, stream);
    }
    int bn = 16;
    while (bn < mean && bn < bn_max) bn *= 2;
    if (!byte_map(&m.x, x, a.P, row_bytes, x_pitch, bn) || !byte_map(&m.w0, w0, wrows, row_bytes, row_bytes, kLanes) ||
        !byte_map(&m.w1, glu ? w1 : w0, wrows, row_bytes, row_bytes, kLanes))
        return set_error(VQMOE_LAUNCH_FAILED, "grouped product: tensor map");
    const long long tok_tiles = a.off ? std::min<long long>(a.P, (long long)a.P / bn + groups) : (a.P + bn - 1) / bn;
    const long long ntiles = (a.N + kLanes - 1) / kLanes;
    const int tiles = (int)std::min<long long>(tok_tiles * ntiles, 1 << 20);
    // few tiles: clusters share a tile's blocks, two blocks a CTA at least
    a.split = 1;
    while (a.split < 8 && (long long)tiles * a.split * 2 <= sm_count() && a.split * 4 <= a.KB) a.split *= 2;
    const int wf = pdl_weights && !a.off;
    if (glu) {
        switch (bn) {
            case 16: return launch_n2<16, 2, true>(m, a, tiles, wf, stream);
            case 32: return launch_n2<32, 2, true>(m, a, tiles, wf, stream);
            default: return launch_n2<64, 2, true>(m, a, tiles, wf, stream);
        }
    }
    if (fp8) {
        switch (bn) {
            case 16: return launch_n2<16, 1, true>(m, a, tiles, wf, stream);
            case 32: return launch_n2<32, 1, true>(m, a, tiles, wf, stream);
            case 64: return launch_n2<64, 1, true>(m, a, tiles, wf, stream);
            default: return launch_n2<128, 1, true>(m, a, tiles, wf, stream);
        }
    }
    switch (bn) {
        case 16: return launch_n2<16, 1, false>(m, a, tiles, wf, stream);
        case 32: return launch_n2<32, 1, false>(m, a, tiles, wf, stream);
        case 64: return launch_n2<64, 1, false>(m, a, tiles, wf, stream);
        default: return launch_n2<128, 1, false>(m, a, tiles, wf, stream);
    }
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
