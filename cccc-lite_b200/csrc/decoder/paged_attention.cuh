// Attention over a cache in pages: the host side that its kernels share.
#pragma once

#include "paged.cuh"

namespace b200
{

// paged_cache.cu: the checked descriptors; false where something is not taken
bool make_paged_cache(int dtype, const cuda_b200_pages* c, PagedCache* p);
bool make_paged_batch(const cuda_b200_batch* b, PagedBatch* p);

// The kernels' segments: packed query rows, CTAs per SM.
constexpr unsigned int kPagedPlainRows = 4, kPagedPlainCtas = 4, kPagedRowsRows = 16;

// paged_rows.cu: `ctas` CTAs at most, one per SM
int launch_paged_rows(PagedParams& p, bool coded, unsigned int ctas, cudaStream_t stream, bool pdl);

}    // namespace b200
