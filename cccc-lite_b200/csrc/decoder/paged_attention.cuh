// Attention over a cache in pages: the host side that its kernels share.
#pragma once

#include "paged.cuh"

namespace b200
{

// paged_cache.cu: the checked descriptors; false where something is not taken
bool make_paged_cache(int dtype, const cuda_b200_pages* c, PagedCache* p);
bool make_paged_batch(const cuda_b200_batch* b, PagedBatch* p);

}    // namespace b200
