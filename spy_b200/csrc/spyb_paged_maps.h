// Tensor maps of caches in pages.
#pragma once

#include <cuda.h>

#include "spyb_paged.cuh"

namespace spyb {

// Pages of bytes, [page][head][position][element] whatever the order of the strides: boxes of `box` positions x all bytes of a head (64 or 128), in the swizzle of as many bytes; false where it cannot be made
bool paged_byte_map(CUtensorMap *map, const void *pool, const PagedView &v, int heads, int head_dim, int box);

}  // namespace spyb
