// Attention over a cache in pages: parameters, E4M3 codes, and what the kernels share on the device.
#pragma once

#include "decoder_common.cuh"
#include "paged_plan.cuh"

namespace b200
{

struct PagedParams : PagedPlan
{
    const void* q;
    void* out;
    const float* sink;
    PagedHeader* header;    // per CTA
    float* partial;         // per CTA two pieces: one of a segment begun before, one of the segment left unfinished
    unsigned int ldq, ldo, H;
    float scale;
};

__host__ __device__ constexpr unsigned int paged_ld(unsigned int vdim) { return (vdim + 15) / 16 * 16; }
// Floats of a piece: values [rows][paged_ld], then maximum and sum of each row.
__host__ __device__ constexpr size_t paged_piece(unsigned int rows, unsigned int vdim) { return (size_t)rows * (paged_ld(vdim) + 2); }

// 2^(b - 127); b in 1 .. 254
__device__ __forceinline__ float paged_two(unsigned int b) { return __uint_as_float(b << 23); }
// Two E4M3 codes as FP16 (exact).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two)
{
    uint32_t r;
    asm("{\n\t.reg .b16 lo;\n\tcvt.u16.u32 lo, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
// Four codes: the lower two, the upper two.
__device__ __forceinline__ void e4m3x4_to_f16x2(uint32_t four, uint32_t& a, uint32_t& b)
{
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(a), "=r"(b) : "r"(four));
}
__device__ __forceinline__ float paged_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// All of the CTA's THREADS threads; `warps` is shared memory for THREADS / 32 sums, `share` is shared too.
template <unsigned int UNIT, unsigned int ROWS, unsigned int THREADS>
__device__ __forceinline__ void paged_share(const PagedParams& p, unsigned long long* warps, PagedShare* share)
{
    const unsigned int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned int per = (p.b.entries + THREADS - 1) / THREADS, e_begin = threadIdx.x * per, e_end = min(e_begin + per, p.b.entries);
    unsigned long long mine = 0;
    for (unsigned int e = e_begin; e < e_end; e++) { mine += paged_head_units<UNIT, ROWS>(p, paged_entry(p, p.b.e0 + e)) * p.c.Hkv; }
    unsigned long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const unsigned long long x = __shfl_up_sync(0xFFFFFFFFu, sum, o);
        if (lane >= (unsigned int)o) { sum += x; }
    }
    if (lane == 31) { warps[warp] = sum; }
    __syncthreads();
    unsigned long long before = 0, total = 0;
#pragma unroll
    for (unsigned int w = 0; w < THREADS / 32; w++)
    {
        if (w < warp) { before += warps[w]; }
        total += warps[w];
    }
    before += sum - mine;
    const unsigned int ctas = paged_ctas(total, p.least, gridDim.x);
    const unsigned long long begin = paged_begin(total, blockIdx.x, ctas), end = paged_begin(total, blockIdx.x + 1, ctas);
    if (threadIdx.x == 0)
    {
        share->total = total;
        share->begin = begin;
        share->end = end;
        share->ctas = ctas;
    }
    if (begin >= before && begin < before + mine && begin < end) { paged_find<UNIT, ROWS>(p, p.b.e0 + e_begin, p.b.e0 + e_end, begin - before, share); }
    __syncthreads();
}

template <class T>
__device__ __forceinline__ void paged_store4(T* out, unsigned int d, unsigned int vdim, bool vec, float4 v)
{
    if (vec) { store4(out + d, v); }
    else
    {
        const float x[4] = { v.x, v.y, v.z, v.w };
        for (unsigned int j = 0; j < 4 && d + j < vdim; j++) { out[d + j] = Elem<T>::put(x[j]); }
    }
}
template <class T>
__device__ __forceinline__ bool paged_vec4(const PagedParams& p)
{
    return (p.c.vdim % 4) == 0 && (p.ldo % 4) == 0 && (reinterpret_cast<uintptr_t>(p.out) % (4 * sizeof(T))) == 0;
}
// The factor that turns weighted values, relative to the maximum m (in powers of two), into the row's output.
__device__ __forceinline__ float paged_factor(const PagedParams& p, unsigned int head, float m, float l)
{
    if (m == -INFINITY && l == 0.f) { return 0.f; }
    if (p.sink != nullptr) { l += paged_exp2(fmaf(p.sink[head], 1.44269504088896341f, -m)); }
    return 1.0f / l;
}

}    // namespace b200
