// TMA tensor maps of the library's tensors.
#pragma once
#include <cuda.h>

#include <cstdint>

namespace vb {
// A 4-D map over a bf16 (or, with f16 set, float16) [B, T, H, D] array: boxes of 64 channels x 1 head x 64 tokens x 1 row,
// 128-byte swizzle (the tiles' shared-memory layout), zero fill outside the array (past T, past D).
int make_token_map(CUtensorMap* map, const void* base, int B, int T, int H, int D, bool f16 = false);
// A 2-D map over `rows` rows of `width` bytes, `pitch` bytes apart: boxes of 128 bytes x box_rows rows, 128-byte
// swizzle, zero fill outside the array.
int make_byte_map(CUtensorMap* map, const void* base, int64_t rows, int64_t width, int64_t pitch, int box_rows);
// A 2-D map for stores into a dense [rows, width] array of 2- or 4-byte elements (`dtype`'s size): boxes of box_width
// elements (128 bytes) x box_rows rows, 128-byte swizzle; what lies outside the array is not stored.
int make_out_map(CUtensorMap* map, void* base, int64_t rows, int64_t width, int box_width, int box_rows, int dtype);
}  // namespace vb
