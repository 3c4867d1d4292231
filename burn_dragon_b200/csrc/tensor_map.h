// tensor_map.h — TMA tensor maps over bf16 memory, encoded in gemm_host.cu.
#pragma once
#include <cuda.h>

#include <array>
#include <cstdint>

namespace bd {

// A map of `dims` (inner, rows, batches) values with `strides` (row, batch) in values, boxes of
// box_inner x box_rows, 128-byte swizzle. Elements outside `dims` read as zero and are not written.
CUtensorMap tensor_map_bf16(const void* base, std::array<int64_t, 3> dims, std::array<int64_t, 2> strides,
                            uint32_t box_inner, uint32_t box_rows);

}  // namespace bd
