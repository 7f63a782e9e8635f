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
    float* partial;         // per worker two pieces: one of a segment begun before, one of the segment left unfinished
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

// Where the units of the entries lie, in shared memory: before[i] units come before those of thread i's entries, before[THREADS] are all.
template <unsigned int THREADS>
struct PagedSums
{
    unsigned long long before[THREADS + 1], warps[THREADS / 32];
};
// By all of the CTA's THREADS threads.
template <unsigned int UNIT, unsigned int ROWS, unsigned int THREADS>
__device__ __forceinline__ void paged_sums(const PagedParams& p, PagedSums<THREADS>* s)
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
    if (lane == 31) { s->warps[warp] = sum; }
    __syncthreads();
    unsigned long long before = 0;
#pragma unroll
    for (unsigned int w = 0; w < THREADS / 32; w++) { before += w < warp ? s->warps[w] : 0; }
    s->before[threadIdx.x] = before + sum - mine;
    if (threadIdx.x == THREADS - 1) { s->before[THREADS] = before + sum; }
    __syncthreads();
}
// The share of one of `most` workers; by any thread, after paged_sums.
template <unsigned int UNIT, unsigned int ROWS, unsigned int THREADS>
__device__ __forceinline__ PagedShare paged_share(const PagedParams& p, const PagedSums<THREADS>& s, unsigned int worker, unsigned int most)
{
    PagedShare x = {};
    x.total = s.before[THREADS];
    x.workers = paged_workers(x.total, p.least, most);
    x.begin = paged_begin(x.total, worker, x.workers);
    x.end = paged_begin(x.total, worker + 1, x.workers);
    if (x.begin >= x.end) { return x; }
    unsigned int lo = 0, hi = THREADS;    // before[lo] <= begin < before[hi]
    while (hi - lo > 1)
    {
        const unsigned int mid = (lo + hi) / 2;
        if (s.before[mid] <= x.begin) { lo = mid; }
        else { hi = mid; }
    }
    const unsigned int per = (p.b.entries + THREADS - 1) / THREADS;
    paged_find<UNIT, ROWS>(p, p.b.e0 + lo * per, p.b.e0 + min((lo + 1) * per, p.b.entries), x.begin - s.before[lo], &x);
    return x;
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

// A warp puts four neighbouring rows of pieces together, eight lanes a row: lane s of them has the elements 32 k + 4 s .. of k < K.
template <int K>
struct PagedQuad
{
    float top, sum;
    float4 acc[K];
};
// Rows r .. r + 3 (those below `end`) of `n` pieces, up to eight, in their order: the first one, then those at `others`, `step` floats from
// one to the next.  Everything that is asked for is under way at once.
template <int K>
__device__ __forceinline__ PagedQuad<K> paged_join(const float* first, const float* others, size_t step, unsigned int n, unsigned int r, unsigned int end, unsigned int VL,
    unsigned int rows)
{
    const unsigned int lane = threadIdx.x & 31, s = lane & 7u, row = r + (lane >> 3);
    const bool real = row < end;
    auto at = [&](unsigned int j) { return j == 0 ? first : others + (size_t)(j - 1) * step; };
    const float m = real && s < n ? at(s)[rows * VL + row] : -INFINITY, l = real && s < n ? at(s)[rows * VL + rows + row] : 0.f;
    constexpr unsigned int B = K <= 4 ? 4 : 2;    // pieces at a time
    float4 y[B][K];
    auto fetch = [&](unsigned int j0) {
#pragma unroll
        for (unsigned int j = 0; j < B; j++)
        {
#pragma unroll
            for (unsigned int k = 0; k < K; k++)
            {
                y[j][k] = real && j0 + j < n && k * 32 + s * 4 < VL ? load4(at(j0 + j) + (size_t)row * VL + k * 32 + s * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    };
    fetch(0);
    PagedQuad<K> x;
    x.top = m;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) { x.top = fmaxf(x.top, __shfl_xor_sync(0xFFFFFFFFu, x.top, o)); }
    const float f = s >= n ? 0.f : x.top == -INFINITY ? 1.f : exp2f(m - x.top);
    x.sum = f * l;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) { x.sum += __shfl_xor_sync(0xFFFFFFFFu, x.sum, o); }
#pragma unroll
    for (unsigned int k = 0; k < K; k++) { x.acc[k] = make_float4(0.f, 0.f, 0.f, 0.f); }
    for (unsigned int j0 = 0; j0 < n; j0 += B)
    {
        if (j0 != 0) { fetch(j0); }
#pragma unroll
        for (unsigned int j = 0; j < B; j++)
        {
            const float w = __shfl_sync(0xFFFFFFFFu, f, (lane & 24u) + ((j0 + j) & 7u));
#pragma unroll
            for (unsigned int k = 0; k < K; k++)
            {
                x.acc[k] = make_float4(fmaf(w, y[j][k].x, x.acc[k].x), fmaf(w, y[j][k].y, x.acc[k].y), fmaf(w, y[j][k].z, x.acc[k].z), fmaf(w, y[j][k].w, x.acc[k].w));
            }
        }
    }
    return x;
}
// Row r + lane / 8 of a segment (its packed row `row`, of those below `end`) as an output.
template <class T, int K>
__device__ __forceinline__ void paged_put(const PagedParams& p, const PagedQuad<K>& x, unsigned int start, unsigned int kvh, unsigned int row, bool real)
{
    if (!real) { return; }
    const unsigned int s = threadIdx.x & 7u, head = kvh * p.G + row % p.G;
    const float f = paged_factor(p, head, x.top, x.sum);
    const bool vec = paged_vec4<T>(p);
    T* out = (T*)p.out + (size_t)(start + row / p.G) * p.ldo + (size_t)head * p.c.vdim;
#pragma unroll
    for (unsigned int k = 0; k < K; k++)
    {
        const unsigned int d = k * 32 + s * 4;
        if (d < p.c.vdim) { paged_store4(out, d, p.c.vdim, vec, make_float4(x.acc[k].x * f, x.acc[k].y * f, x.acc[k].z * f, x.acc[k].w * f)); }
    }
}

}    // namespace b200
