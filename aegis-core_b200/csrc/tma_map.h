#pragma once
// TMA tensor-map encoding for 16-bit and 8-bit operands (cuTensorMapEncodeTiled through
// the runtime's driver entry point, so the library needs no libcuda link).
#include <cuda.h>

#include "aegis/gemm.h"

namespace aegis {

// A 3-D (inner, outer, batch) 16-bit tensor with 128-byte-swizzled boxes of
// {64, box_outer, 1}; ld and batch stride in elements. batch <= 1: the batch
// coordinate is unused. False if the driver refuses the geometry.
bool encode_map(CUtensorMap* map, gemm::DType dt, const void* base, long long inner, long long outer, long long ld,
                long long batch, long long bstride, int box_outer);

// The same for rows of 8-bit codes, ld in bytes (a multiple of 16, as is the base
// address). blocks = 0: boxes of {128, box_outer, 1}. blocks > 0, inner a multiple
// of 128: the rows as (128, outer, inner / 128), boxes of {128, box_outer, blocks}.
bool encode_map_i8(CUtensorMap* map, const void* base, long long inner, long long outer, long long ld, int box_outer,
                   int blocks = 0);

}  // namespace aegis
