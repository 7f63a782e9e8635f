// Attention over a cache in pages: the entry point, the plain kernel (any sizes and types, and the float mode), and the kernel that
// puts the pieces of segments together which more than one CTA has worked on.
#include "paged_attention.cuh"

namespace b200
{

// ---- plain kernel ------------------------------------------------------------------------------------------------
// Four packed query rows per segment, units of 32 keys, one key per lane for the scores and one element per lane for the values.
// The warps of a CTA take the units in turn, each with its own maximum and sum.
constexpr unsigned int PP_UNIT = 32, PP_ROWS = kPagedPlainRows, PP_WARPS = 4, PP_THREADS = 32 * PP_WARPS, PP_ELEMS = 8;    // elements of a value row per lane

template <class C>
__device__ __forceinline__ float4 cache4(const C* p) { return load4(p); }
template <>
__device__ __forceinline__ float4 cache4(const unsigned char* p)
{
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p), a = e4m3x2_to_f16x2(w), b = e4m3x2_to_f16x2(w >> 16);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    return make_float4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ float cache1(const float* p) { return *p; }
__device__ __forceinline__ float cache1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float cache1(const unsigned char* p)
{
    const uint32_t a = e4m3x2_to_f16x2(*p);
    return __low2float(*reinterpret_cast<const __half2*>(&a));
}

template <class T, class C>
__global__ void __launch_bounds__(PP_THREADS) paged_plain_kernel(const __grid_constant__ PagedParams p)
{
    constexpr bool CODED = sizeof(C) == 1;
    __shared__ PagedShare share;
    __shared__ unsigned long long sums[PP_WARPS];
    __shared__ __align__(16) float q[PP_ROWS][256];
    __shared__ float acc_s[PP_WARPS][PP_ROWS][32 * PP_ELEMS];
    __shared__ float max_s[PP_WARPS][PP_ROWS], sum_s[PP_WARPS][PP_ROWS];
    const unsigned int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dependency_launch();
    grid_dependency_wait();
    paged_share<PP_UNIT, PP_ROWS, PP_THREADS>(p, sums, &share);
    PagedHeader header = {};
    PagedCursor<PP_UNIT, PP_ROWS> cur;
    unsigned long long at = share.begin;
    if (at < share.end) { cur.at(p, share); }
    while (at < share.end)
    {
        const PagedSegment& s = cur.s;
        const unsigned int units = cur.take(share.end - at);
        for (unsigned int i = threadIdx.x; i < PP_ROWS * 256; i += PP_THREADS)
        {
            const unsigned int r = i / 256, d = i % 256, row = s.r0 + r;
            q[r][d] = r < s.rows && d < p.c.dim
                ? Elem<T>::get(((const T*)p.q)[(size_t)(cur.v.start + row / p.G) * p.ldq + (size_t)(cur.kvh * p.G + row % p.G) * p.c.dim + d]) : 0.f;
        }
        __syncthreads();
        float m[PP_ROWS], l[PP_ROWS], acc[PP_ROWS][PP_ELEMS];
#pragma unroll
        for (unsigned int r = 0; r < PP_ROWS; r++)
        {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (unsigned int i = 0; i < PP_ELEMS; i++) { acc[r][i] = 0.f; }
        }
        for (unsigned int u = warp; u < units; u += PP_WARPS)
        {
            const unsigned int key = s.unit(cur.unit + u) * PP_UNIT + lane;
            const int page = paged_wanted(cur.v, s, key) ? paged_page(p.c, cur.v.slot, key) : -1;
            const size_t row = page < 0 ? 0 : paged_row(p.c, page, cur.kvh, key);
            float z[PP_ROWS] = {};
            float sv = 1.f;
            if (page >= 0)
            {
                const C* k = (const C*)p.c.k + row * p.c.k_ld;
                for (unsigned int d = 0; d < p.c.dim; d += 4)    // the rows are padded with zeros
                {
                    const float4 x = cache4(k + d);
#pragma unroll
                    for (unsigned int r = 0; r < PP_ROWS; r++)
                    {
                        const float4 y = *reinterpret_cast<const float4*>(&q[r][d]);
                        z[r] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, z[r]))));
                    }
                }
                float scale = p.scale * 1.44269504088896341f;
                if constexpr (CODED)
                {
                    scale *= paged_two(p.c.k_scale[row]);
                    sv = paged_two(p.c.v_scale[row]);
                }
#pragma unroll
                for (unsigned int r = 0; r < PP_ROWS; r++) { z[r] *= scale; }
            }
            unsigned int seen[PP_ROWS], any = 0;
            float w[PP_ROWS];
#pragma unroll
            for (unsigned int r = 0; r < PP_ROWS; r++)
            {
                const bool mine = page >= 0 && r < s.rows && paged_seen(p, cur.v, cur.v.pos + (s.r0 + r) / p.G, key);
                seen[r] = __ballot_sync(0xFFFFFFFFu, mine);
                any |= seen[r];
                float top = mine ? z[r] : -INFINITY;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o)); }
                if (top > m[r])
                {
                    const float c = exp2f(m[r] - top);    // 0 where nothing came before
                    m[r] = top;
                    l[r] *= c;
#pragma unroll
                    for (unsigned int i = 0; i < PP_ELEMS; i++) { acc[r][i] *= c; }
                }
                w[r] = mine ? exp2f(z[r] - (m[r] == -INFINITY ? 0.f : m[r])) : 0.f;
                l[r] += warp_sum(w[r]);
                w[r] *= sv;
            }
            const C* v = (const C*)p.c.v + row * p.c.v_ld;
            for (; any != 0; any &= any - 1)
            {
                const int j = __ffs(any) - 1;
                const C* vj = (const C*)__shfl_sync(0xFFFFFFFFu, (unsigned long long)v, j);
                float x[PP_ELEMS];
#pragma unroll
                for (unsigned int i = 0; i < PP_ELEMS; i++) { x[i] = lane + 32 * i < p.c.vdim ? cache1(vj + lane + 32 * i) : 0.f; }
#pragma unroll
                for (unsigned int r = 0; r < PP_ROWS; r++)
                {
                    const float wj = __shfl_sync(0xFFFFFFFFu, w[r], j);
                    if ((seen[r] >> j & 1u) == 0) { continue; }    // a value that is not seen may be no number
#pragma unroll
                    for (unsigned int i = 0; i < PP_ELEMS; i++) { acc[r][i] = fmaf(wj, x[i], acc[r][i]); }
                }
            }
        }
#pragma unroll
        for (unsigned int r = 0; r < PP_ROWS; r++)
        {
            if (lane == 0)
            {
                max_s[warp][r] = m[r];
                sum_s[warp][r] = l[r];
            }
#pragma unroll
            for (unsigned int i = 0; i < PP_ELEMS; i++) { acc_s[warp][r][lane + 32 * i] = acc[r][i]; }
        }
        __syncthreads();
        const bool whole = cur.whole(units);
        const unsigned int VL = paged_ld(p.c.vdim);
        float* piece = p.partial + (2 * (size_t)blockIdx.x + (cur.unit == 0 ? 1 : 0)) * paged_piece(PP_ROWS, p.c.vdim);
        for (unsigned int i = threadIdx.x; i < s.rows * VL; i += PP_THREADS)
        {
            const unsigned int r = i / VL, d = i % VL;
            float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
            for (unsigned int x = 0; x < PP_WARPS; x++) { top = fmaxf(top, max_s[x][r]); }
#pragma unroll
            for (unsigned int x = 0; x < PP_WARPS; x++)
            {
                const float c = top == -INFINITY ? 1.f : exp2f(max_s[x][r] - top);
                sum = fmaf(c, sum_s[x][r], sum);
                o = fmaf(c, acc_s[x][r][d], o);
            }
            if (whole)
            {
                const unsigned int row = s.r0 + r, head = cur.kvh * p.G + row % p.G;
                if (d < p.c.vdim)
                {
                    ((T*)p.out)[(size_t)(cur.v.start + row / p.G) * p.ldo + (size_t)head * p.c.vdim + d] = Elem<T>::put(o * paged_factor(p, head, top, sum));
                }
            }
            else
            {
                piece[i] = o;
                if (d == 0)
                {
                    piece[PP_ROWS * VL + r] = top;
                    piece[PP_ROWS * VL + PP_ROWS + r] = sum;
                }
            }
        }
        __syncthreads();
        if (!whole && cur.unit == 0) { header = cur.header(share, at, blockIdx.x); }
        at += units;
        if (at < share.end) { cur.next(p); }
    }
    if (threadIdx.x == 0) { p.header[blockIdx.x] = header; }
}

// ---- pieces together ---------------------------------------------------------------------------------------------
// A warp per row: the segment that CTA x left unfinished, its own piece and the first ones of the CTAs behind it.
template <class T, unsigned int ROWS>
__global__ void __launch_bounds__(128) paged_combine_kernel(const __grid_constant__ PagedParams p)
{
    grid_dependency_launch();
    grid_dependency_wait();
    const PagedHeader h = p.header[blockIdx.x];
    if (h.entry == 0) { return; }
    const unsigned int lane = threadIdx.x & 31, r = blockIdx.y * 4 + (threadIdx.x >> 5), VL = paged_ld(p.c.vdim);
    const PagedEntry v = paged_entry(p, h.entry - 1);
    const unsigned int row = h.rt * ROWS + r;
    if (row >= v.n * p.G) { return; }
    const size_t size = paged_piece(ROWS, p.c.vdim);
    auto piece = [&](unsigned int i) { return p.partial + (2 * (size_t)(blockIdx.x + i) + (i == 0 ? 1 : 0)) * size; };
    float top = -INFINITY;
    for (unsigned int i = lane; i < h.pieces; i += 32) { top = fmaxf(top, piece(i)[ROWS * VL + r]); }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o)); }
    float sum = 0.f;
    float4 acc[2] = { make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f) };
#pragma unroll 4
    for (unsigned int i = 0; i < h.pieces; i++)
    {
        const float* x = piece(i);
        const float c = top == -INFINITY ? 1.f : exp2f(x[ROWS * VL + r] - top);
        sum = fmaf(c, x[ROWS * VL + ROWS + r], sum);
#pragma unroll
        for (unsigned int k = 0; k < 2; k++)
        {
            const unsigned int d = lane * 4 + k * 128;
            if (d < VL)
            {
                const float4 y = load4(x + (size_t)r * VL + d);
                acc[k].x = fmaf(c, y.x, acc[k].x);
                acc[k].y = fmaf(c, y.y, acc[k].y);
                acc[k].z = fmaf(c, y.z, acc[k].z);
                acc[k].w = fmaf(c, y.w, acc[k].w);
            }
        }
    }
    const unsigned int head = h.kvh * p.G + row % p.G;
    const float f = paged_factor(p, head, top, sum);
    T* out = (T*)p.out + (size_t)(v.start + row / p.G) * p.ldo + (size_t)head * p.c.vdim;
    const bool vec = paged_vec4<T>(p);
#pragma unroll
    for (unsigned int k = 0; k < 2; k++)
    {
        const unsigned int d = lane * 4 + k * 128;
        if (d < p.c.vdim) { paged_store4(out, d, p.c.vdim, vec, make_float4(acc[k].x * f, acc[k].y * f, acc[k].z * f, acc[k].w * f)); }
    }
}

template <class T, unsigned int ROWS>
static int combine(const PagedParams& p, unsigned int rows, unsigned int ctas, cudaStream_t stream)
{
    return launch_kernel("paged_combine", paged_combine_kernel<T, ROWS>, dim3(ctas, (rows + 3) / 4), dim3(128), 0, stream, true, p);
}

// ---- dispatch ----------------------------------------------------------------------------------------------------
// Scratch: a header for each CTA of the kernel that has most of them, then the pieces.
static size_t header_bytes(unsigned int sms) { return (size_t)sms * kPagedPlainCtas * sizeof(PagedHeader); }
static size_t work_of(unsigned int sms, unsigned int ctas_per_sm, unsigned int rows, unsigned int vdim)
{
    return header_bytes(sms) + 2 * (size_t)sms * ctas_per_sm * paged_piece(rows, vdim) * 4;
}

template <class T, class C>
static int run_plain(PagedParams& p, unsigned int rows, unsigned int ctas, cudaStream_t stream, bool pdl)
{
    p.least = 2 * PP_WARPS;
    const int rc = launch_kernel("paged_plain", paged_plain_kernel<T, C>, dim3(ctas), dim3(PP_THREADS), 0, stream, pdl, p);
    return rc ? rc : combine<T, PP_ROWS>(p, rows < PP_ROWS ? rows : PP_ROWS, ctas, stream);
}

}    // namespace b200

using namespace b200;

C_EXPORT unsigned long long cuda_b200_paged_attention_work_bytes(unsigned int H, unsigned int Hkv, unsigned int vdim, unsigned int max_n)
{
    const DecoderDevice* dev = decoder_device();
    if (!dev || Hkv == 0 || H == 0 || (H % Hkv) || vdim == 0 || vdim > 256 || (unsigned long long)max_n * (H / Hkv) > 0x7FFFFFFFull) { return 0; }
    // the plain kernel and the one for few rows take the same
    static_assert(kPagedPlainCtas * kPagedPlainRows == kPagedRowsRows, "");
    return work_of(dev->sm_count, 1, kPagedRowsRows, vdim);
}

C_EXPORT int cuda_b200_paged_attention_rows(int dtype, const cuda_b200_paged_attention* a, const cuda_b200_pages* c, const cuda_b200_batch* b, void* stream,
    unsigned int flags, int kernel)
{
    if (!a || !b) { return -1; }
    if (b->tokens == 0 || b->entries == 0 || b->max_n == 0) { return 0; }
    PagedParams p;
    if (!a->q || !a->out || !a->work || !make_paged_cache(dtype, c, &p.c) || !make_paged_batch(b, &p.b)) { return -1; }
    if (a->H == 0 || (a->H % c->Hkv) || a->ldq < (unsigned long long)a->H * c->dim || a->ldo < (unsigned long long)a->H * c->vdim
        || (unsigned long long)b->max_n * (a->H / c->Hkv) > 0x7FFFFFFFull || (reinterpret_cast<uintptr_t>(a->work) & 15u) || kernel < 0 || kernel > 2)
    {
        return -1;
    }
    const DecoderDevice* dev = decoder_device();
    if (!dev) { return 1; }
    p.q = a->q;
    p.out = a->out;
    p.sink = (const float*)a->sink;
    p.header = (PagedHeader*)a->work;
    p.partial = (float*)((unsigned char*)a->work + header_bytes(dev->sm_count));
    p.ldq = a->ldq;
    p.ldo = a->ldo;
    p.H = a->H;
    p.G = a->H / c->Hkv;
    p.window = a->window;
    p.first = a->first;
    p.scale = a->scale;
    const bool pdl = (flags & 1u) != 0, coded = c->type == DT_E4M3;
    const cudaStream_t st = (cudaStream_t)stream;
    const unsigned int rows = b->max_n * p.G, sms = (unsigned int)dev->sm_count;
    if (a->work_bytes < work_of(sms, 1, kPagedRowsRows, c->vdim)) { return -1; }
    if (dtype == DT_FLOAT) { kernel = 1; }
    if (kernel == 0) { kernel = 2; }
    if (kernel == 2)
    {
        const int rc = launch_paged_rows(p, coded, rows, sms, st, pdl);
        if (rc) { return rc; }
        return rows <= 8 ? combine<__nv_bfloat16, 8>(p, rows, sms, st) : combine<__nv_bfloat16, kPagedRowsRows>(p, rows < kPagedRowsRows ? rows : kPagedRowsRows, sms, st);
    }
    const unsigned int ctas = sms * kPagedPlainCtas;
    if (dtype == DT_FLOAT) { return coded ? run_plain<float, unsigned char>(p, rows, ctas, st, pdl) : run_plain<float, float>(p, rows, ctas, st, pdl); }
    return coded ? run_plain<__nv_bfloat16, unsigned char>(p, rows, ctas, st, pdl) : run_plain<__nv_bfloat16, __nv_bfloat16>(p, rows, ctas, st, pdl);
}
