// Attention over a cache in pages: the host side that its kernels share.
#pragma once

#include "../tensor_map.cuh"
#include "paged.cuh"

namespace b200
{

// paged_cache.cu: the checked descriptors; false where something is not taken
bool make_paged_cache(int dtype, const cuda_b200_pages* c, PagedCache* p);
bool make_paged_batch(const cuda_b200_batch* b, PagedBatch* p);

// A cache's rows as [pages][Hkv * page][ld], copied `rows` at a time in pieces of `cols` elements.
inline bool make_paged_map(CUtensorMap* map, bool coded, const void* base, unsigned int ld, const PagedCache& c, unsigned int cols, unsigned int rows, bool swizzle)
{
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn || c.pages == 0) { return false; }
    const cuuint64_t bytes = (cuuint64_t)ld * (coded ? 1 : 2), of_page = (cuuint64_t)c.Hkv << c.shift;
    const cuuint64_t dims[3] = { ld, of_page, c.pages }, strides[2] = { bytes, bytes * of_page };
    const cuuint32_t box[3] = { cols, rows, 1 }, one[3] = { 1, 1, 1 };
    return fn(map, coded ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
        == CUDA_SUCCESS;
}

// Has the kernel been given this many registers a thread?  A split of them at run time that adds up to more would wait for good.
template <class K>
inline bool paged_registers(K kernel, int least)
{
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kernel) == cudaSuccess && a.numRegs >= least;
}

// The plain kernel: packed query rows of a segment, CTAs per SM.  The one for few rows (8 or 16 of them): warps of an SM that take shares.
constexpr unsigned int kPagedPlainRows = 4, kPagedPlainCtas = 4, kPagedRowsWarps = 8;
// Packed query rows of an entry up to which that one is taken.
constexpr unsigned int kPagedFewRows = 16;

// paged_rows.cu: a CTA on each of `sms` SMs; *per: its workers
int launch_paged_rows(PagedParams& p, bool coded, unsigned int rows, unsigned int sms, unsigned int* per, cudaStream_t stream, bool pdl);

// paged_tile.cu: a CTA on each SM; *piece_rows: packed query rows of a segment
int launch_paged_tile(PagedParams& p, bool coded, unsigned int sms, unsigned int* piece_rows, cudaStream_t stream, bool pdl);

}    // namespace b200
