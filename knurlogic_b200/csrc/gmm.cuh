// Products of token rows with the weights of their group (an expert, or the
// one group of a dense linear), on tcgen05: block-scaled e4m3 or bf16.
#pragma once

#include "common.cuh"

namespace vqmoe {

constexpr int kScaleBlock = 128;      // inputs (and weight rows) of one float32 scale
constexpr int kMaxGroups = 1024;

// Bytes of a row are cut into KB blocks of 128 (the last one ragged): 128
// e4m3 inputs, one scale block, or 64 bf16 inputs.
struct GmmArgs {
    const int32_t *off;               // [E + 1] device offsets of the groups' rows; null: one group of P rows
    int E, P;                         // groups, rows of x
    int N, KB;                        // output features of a group, 128-byte blocks of a row
    const float *sx;                  // e4m3: token scales, block-major [KB][P]
    const float *sw0, *sw1;           // e4m3: weight scales [E][ceil(N / 128)][KB]
    void *out;                        // [rows][out_stride] bf16 or float32 (null with q_out)
    long long out_stride;
    int out_f32;
    const int32_t *map;               // row -> output row; null: the row itself
    const float *row_scale;           // optional, by output row: bf16(bf16(y) * s)
    uint8_t *q_out;                   // gate/up: the activations quantized, e4m3 [P][N] ...
    float *s_out;                     // ... and their scales, block-major [ceil(N / 128)][P]
    int act;                          // gate/up: VQMOE_ACT_*
    uint32_t *err;                    // word raised when a bounded wait ran out, or null
};

// x: rows of `row_bytes` bytes at a pitch of x_pitch bytes; w0 (and w1, the
// up matrix of a fused gate/up): [E * N] rows of row_bytes. fp8 false: bf16.
// pdl_weights: the weights may be read before the kernel's predecessor on the
// stream has finished (nothing queued may still write them).
vqmoe_status launch_gmm(const void *x, size_t x_pitch, const void *w0, const void *w1, size_t row_bytes, bool fp8,
                        const GmmArgs &a, cudaStream_t stream, bool pdl_weights = false);

// bf16 rows -> e4m3 rows [..][cols] and float32 scales, element (row, g) at
// s[row * s_row + g * s_group]. With `order` the rows of x (one for each of
// order->k pairs) go to their pairs' positions.
struct QuantOrder {
    const int32_t *inds, *rank, *off; // pair -> expert, rank in it; expert -> first position
    int E, k, per_pair;               // k pairs a row, or (per_pair) one
};
vqmoe_status launch_quantize_fp8(const void *x, long long rows, int cols, long long x_stride, uint8_t *q, float *s,
                                 long long s_row, long long s_group, const QuantOrder *order, cudaStream_t stream);

}  // namespace vqmoe
