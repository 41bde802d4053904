// Host side of the TMA tensor copies: tensor maps encoded through the
// driver entry point the CUDA runtime exposes (no link against the driver
// library).
#pragma once

#include <cuda.h>

namespace vqmoe {

// Any row-major 2-D tensor with rows at a pitch of `pitch` bytes (dims and
// box in elements, columns first), 128-byte swizzle; and
// row-major [rows][cols] of 2-byte elements (row pitch cols * 2, a multiple
// of 16; base 16-byte aligned): boxes of box_rows rows x 64 columns (128
// bytes) with the 128-byte swizzle; out-of-range elements read as zero.
CUresult encode_tma_2d(CUtensorMap *m, CUtensorMapDataType type, const void *base, const cuuint64_t (&dims)[2],
                       cuuint64_t pitch, const cuuint32_t (&box)[2]);
bool make_tma_map(CUtensorMap *m, const void *base, int rows, int cols, int box_rows);

}  // namespace vqmoe
