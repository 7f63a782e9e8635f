// Attention of few query rows (up to 16 packed ones per segment: decoding) over a cache in pages, HBM-bound, on mma.sync.
//
// Every warp streams units of its own through a ring in shared memory that only it uses, with cp.async, three deep: a lane later reads
// back just what it has copied, so that no barrier stands between the warps while they stream.  What a lane copies is what
// its fragments need.  Scores: keys are the columns of m16n8k16, a lane holds 16 bytes of its key's row and takes them as the
// k places of several products (the queries' elements are permuted alike).  Values: a lane holds the same 16 bytes of four keys; byte
// permutes pair two keys' elements, and its elements are the same column of several products (the output columns are permuted, and put
// back on store).
//
// E4M3: codes become FP16 by one instruction per pair, exactly.  Queries enter as FP16, each row by a power of two below 2^15
// (exact for elements down to 2^-28 of the row's largest).  A key's power of two multiplies its score.  A value's one, 2^u, goes to the
// weight: with m the maximum of score + u, p = 2^(score - m) counts in the sum and w = p 2^u <= 2^8 in the product, as FP16 - the
// weights are rounded by 2^-12 of each at most, whatever the rows' scales.  BF16: weights enter as the sum of two BF16 numbers.
// The maximum moves only when it grows by more than 2^8, so that the outputs are seldom rescaled.
#include "paged_attention.cuh"

#include "../gemv_decode.cuh"

#include <type_traits>

namespace b200
{

constexpr unsigned int RW_ROWS = 16, RW_STAGES = 3, RW_MERGE = 4;    // rows that the warps put together at a time

template <int D, bool CODED>
struct RowsShape
{
    static constexpr int EB = CODED ? 1 : 2;
    static constexpr int ROW = D * EB;                                  // bytes of a cache row
    static constexpr int WARPS = ROW > 256 ? 4 : 8;
    static constexpr int UNIT = ROW >= 256 ? 16 : 4096 / ROW;           // keys: 8 KB a stage (16 KB for the longest rows)
    static constexpr int SUB = UNIT / 16;
    static constexpr int EPC = 16 / EB;                                 // elements of a 16-byte piece
    static constexpr int KI = ROW / 64;                                 // pieces of a key row per lane: i * 4 + lane % 4
    static constexpr int VB = ROW < 128 ? ROW / 8 : 16;                 // bytes of a value piece
    static constexpr int VI = ROW / (8 * VB);                           // pieces of a value row per lane: i * 8 + lane / 4
    static constexpr int VE = VB / EB;                                  // its elements
    static constexpr int STAGE = 2 * UNIT * ROW;
    static constexpr int SCALES = CODED ? 2 * UNIT : 0;                 // exponent bytes of a stage
    static constexpr int INFO = 16;                                     // of a stage: first key, subtiles on no page
    static constexpr int MERGE_LD = D + 4;
    static constexpr int RING = RW_STAGES * STAGE;
    static constexpr int SMALL = RW_STAGES * (SCALES + INFO);
    static constexpr int SMEM = WARPS * (RING + SMALL) + WARPS * (int)RW_MERGE * MERGE_LD * 4;
};

__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src, uint32_t bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
template <bool F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (F16)
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    else
    {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int D, bool CODED>
__global__ void __launch_bounds__(32 * RowsShape<D, CODED>::WARPS, 1) paged_rows_kernel(const __grid_constant__ PagedParams p)
{
    using S = RowsShape<D, CODED>;
    constexpr unsigned int UNIT = S::UNIT, WARPS = S::WARPS, THREADS = 32 * WARPS;
    constexpr int STEPS = D / 16, TILES = UNIT / 8;
    extern __shared__ __align__(16) unsigned char rw_smem[];
    __shared__ PagedShare share;
    __shared__ unsigned long long sums[WARPS];
    __shared__ PagedCursor<UNIT, RW_ROWS> cur_s;
    __shared__ float max_s[WARPS][RW_ROWS], sum_s[WARPS][RW_ROWS];
    const unsigned int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(rw_smem) + warp * S::RING + lane * 16;
    unsigned char* small = rw_smem + WARPS * S::RING + warp * S::SMALL;    // per stage: info, exponents of keys, of values
    float* merge = reinterpret_cast<float*>(rw_smem + WARPS * (S::RING + S::SMALL));

    grid_dependency_launch();
    grid_dependency_wait();
    paged_share<UNIT, RW_ROWS, THREADS>(p, sums, &share);
    if (share.begin >= share.end)
    {
        if (threadIdx.x == 0) { p.header[blockIdx.x] = PagedHeader{}; }
        return;
    }
    const unsigned long long begin = share.begin, end = share.end;

    // ---- what the warp asks for: units begin + warp, begin + warp + WARPS, ... of the share, across its segments ----
    PagedCursor<UNIT, RW_ROWS> ask;
    unsigned long long ask_at = begin + warp, ask_seg = begin;    // the unit, and where its segment's units in the share begin
    ask.at(p, share);
    unsigned int ask_key = 0;
    int ask_page = -1;    // lane i: the page of the unit's i-th sixteen keys
    auto find = [&]() {
        if (ask_at >= end) { return; }
        for (unsigned int n = ask.s.count - ask.unit; ask_at - ask_seg >= n; n = ask.s.count)
        {
            ask_seg += n;
            ask.next(p);
        }
        ask_key = ask.s.unit(ask.unit + (unsigned int)(ask_at - ask_seg)) * UNIT;
        const unsigned int first = ask_key + lane * 16;
        ask_page = -1;
        // a range of keys meets one of the two wanted ranges
        if (lane < (unsigned int)S::SUB && first < ask.s.lim && (first + 16 > ask.s.low || (first + 16 > ask.v.floor && first < ask.s.first_end)))
        {
            ask_page = paged_page(p.c, ask.v.slot, first);
        }
    };
    const unsigned int kb = p.c.k_ld * S::EB, vb = p.c.v_ld * S::EB;
    auto request = [&](unsigned int stage) {
        if (ask_at < end)
        {
            const uint32_t to = ring + stage * S::STAGE;
            unsigned char* info = small + stage * (S::INFO + S::SCALES);
            const unsigned int bad = __ballot_sync(0xFFFFFFFFu, lane < (unsigned int)S::SUB && ask_page < 0);
            if (lane == 0) { *reinterpret_cast<uint2*>(info) = make_uint2(ask_key, bad); }
            const bool all = bad == 0 && ask_key + UNIT <= ask.s.lim && ask_key >= ask.s.low;
#pragma unroll
            for (int s = 0; s < S::SUB; s++)
            {
                const int page = __shfl_sync(0xFFFFFFFFu, ask_page, s);
                const unsigned int key = ask_key + s * 16;
                const size_t row = page < 0 ? 0 : paged_row(p.c, page, ask.kvh, key);
                auto wanted = [&](unsigned int j) { return all || (page >= 0 && paged_wanted(ask.v, ask.s, key + j)); };
                if constexpr (CODED)
                {
                    if (lane < 2) { cp_async(smem_u32(info) + S::INFO + lane * UNIT + s * 16, (lane ? p.c.v_scale : p.c.k_scale) + row, page < 0 ? 0 : 16); }
                }
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    const unsigned char* src = p.c.k + (row + h * 8 + g) * kb;
                    const bool w = wanted(h * 8 + g);
#pragma unroll
                    for (int i = 0; i < S::KI; i++)
                    {
                        const unsigned int at = (i * 4 + t) * 16;
                        const bool take = w && at < kb;
                        cp_async(to + ((s * 2 + h) * S::KI + i) * 512, take ? src + at : p.c.k, take ? 16u : 0u);
                    }
                }
#pragma unroll
                for (int h = 0; h < 4; h++)
                {
                    const unsigned int j = (h >> 1) * 8 + 2 * t + (h & 1);
                    const unsigned char* src = p.c.v + (row + j) * vb;
                    const bool w = wanted(j);
#pragma unroll
                    for (int i = 0; i < S::VI; i++)
                    {
                        const unsigned int at = (i * 8 + g) * S::VB;
                        const bool take = w && at < vb;
                        const uint32_t dst = to + UNIT * S::ROW + ((s * 4 + h) * S::VI + i) * 32 * S::VB - (S::VB == 8 ? lane * 8 : 0);
                        if constexpr (S::VB == 16) { cp_async(dst, take ? src + at : p.c.v, take ? 16u : 0u); }
                        else { cp_async8(dst, take ? src + at : p.c.v, take ? 8u : 0u); }
                    }
                }
            }
            ask_at += WARPS;
            find();
        }
        cp_async_commit();
    };
    find();
#pragma unroll
    for (unsigned int s = 0; s + 1 < RW_STAGES; s++) { request(s); }
    unsigned int stage = 0;

    if (threadIdx.x == 0) { cur_s.at(p, share); }
    PagedHeader header = {};
    unsigned long long at = begin, mine = begin + warp;    // the segment's first unit; the warp's next unit
    while (at < end)
    {
        __syncthreads();
        const PagedEntry v = cur_s.v;
        const PagedSegment s = cur_s.s;
        const unsigned int kvh = cur_s.kvh, units = cur_s.take(end - at);
        // ---- queries: rows g and g + 8 of the segment ----
        uint32_t q[STEPS][4];
        float rs[2];
        unsigned int tok[2];    // their tokens' positions
#pragma unroll
        for (int h = 0; h < 2; h++)
        {
            const unsigned int r = s.r0 + g + 8 * h;
            const bool real = g + 8 * h < s.rows;
            tok[h] = v.pos + (real ? r / p.G : 0);
            const __nv_bfloat16* src = (const __nv_bfloat16*)p.q + (real ? (size_t)(v.start + r / p.G) * p.ldq + (size_t)(kvh * p.G + r % p.G) * p.c.dim : 0);
            const bool vec = (p.c.dim % 4) == 0 && (p.ldq % 4) == 0 && (reinterpret_cast<uintptr_t>(p.q) % 8) == 0;
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < STEPS; k++)
            {
                const unsigned int d = (k / (S::EPC / 4) * 4 + t) * S::EPC + k % (S::EPC / 4) * 4;
                uint2 u = make_uint2(0, 0);
                if (real && d < p.c.dim)
                {
                    if (vec) { u = *reinterpret_cast<const uint2*>(src + d); }
                    else
                    {
                        uint32_t x[4];
#pragma unroll
                        for (unsigned int j = 0; j < 4; j++) { x[j] = d + j < p.c.dim ? __bfloat16_as_ushort(src[d + j]) : 0u; }
                        u = make_uint2(x[0] | (x[1] << 16), x[2] | (x[3] << 16));
                    }
                }
                q[k][h] = u.x;
                q[k][2 + h] = u.y;
                if constexpr (CODED)
                {
                    top = max(max(top, max((u.x << 16) & 0x7FFF0000u, u.x & 0x7FFF0000u)), max((u.y << 16) & 0x7FFF0000u, u.y & 0x7FFF0000u));
                }
            }
            rs[h] = p.scale * 1.44269504088896341f;
            if constexpr (CODED)
            {
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                // the largest element comes to 2^14 .. 2^15
                const unsigned int b = min(268u - (top >> 23), 254u);
                const float f = paged_two(b);
                rs[h] *= b == 254u ? 5.877471754e-39f : paged_two(254u - b);    // 2^-127 is not a normal number
#pragma unroll
                for (int k = 0; k < STEPS; k++)
                {
#pragma unroll
                    for (int x = h; x < 4; x += 2)
                    {
                        q[k][x] = pack_f16x2(__uint_as_float(q[k][x] << 16) * f, __uint_as_float(q[k][x] & 0xFFFF0000u) * f);
                    }
                }
            }
        }
        float acc[D / 8][4], m[2] = { -INFINITY, -INFINITY }, l[2] = { 0.f, 0.f };
#pragma unroll
        for (int i = 0; i < D / 8; i++) { acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f; }
        // keys that every row sees
        const unsigned int lim_all = min(v.pos + s.r0 / p.G + 1, s.lim), t_last = v.pos + (s.r0 + s.rows - 1) / p.G;
        const unsigned int low_all = max(v.floor, p.window != 0 && t_last + 1 > p.window ? t_last + 1 - p.window : 0u);

        for (; mine < at + units; mine += WARPS)
        {
            cp_async_wait<RW_STAGES - 2>();
            __syncwarp();
            request((stage + RW_STAGES - 1) % RW_STAGES);
            const uint32_t from = ring + stage * S::STAGE;
            unsigned char* info = small + stage * (S::INFO + S::SCALES);
            const uint2 what = *reinterpret_cast<const uint2*>(info);
            // ---- scores ----
            float z[TILES][4];
#pragma unroll
            for (int j = 0; j < TILES; j++) { z[j][0] = z[j][1] = z[j][2] = z[j][3] = 0.f; }
#pragma unroll
            for (int i = 0; i < S::KI; i++)
            {
#pragma unroll
                for (int j = 0; j < TILES; j++)
                {
                    const uint4 k = lds128(from + (j * S::KI + i) * 512);
                    const uint32_t w[4] = { k.x, k.y, k.z, k.w };
                    if constexpr (CODED)
                    {
#pragma unroll
                        for (int x = 0; x < 4; x++) { mma16816<true>(z[j], q[i * 4 + x], e4m3x2_to_f16x2(w[x]), e4m3x2_to_f16x2(w[x] >> 16)); }
                    }
                    else
                    {
                        mma16816<false>(z[j], q[i * 2], w[0], w[1]);
                        mma16816<false>(z[j], q[i * 2 + 1], w[2], w[3]);
                    }
                }
            }
            // ---- weights ----
            uint32_t ev[TILES];    // exponent bytes of a lane's two values
            float top[2] = { -INFINITY, -INFINITY };
            const bool all = what.y == 0 && what.x >= low_all && what.x + UNIT <= lim_all;
#pragma unroll
            for (int j = 0; j < TILES; j++)
            {
                float sk[2] = { 1.f, 1.f };
                if constexpr (CODED)
                {
                    const uint32_t ek = lds_u16(smem_u32(info) + S::INFO + j * 8 + 2 * t);
                    ev[j] = lds_u16(smem_u32(info) + S::INFO + UNIT + j * 8 + 2 * t);
                    sk[0] = paged_two(ek & 255u);
                    sk[1] = paged_two(ek >> 8);
                }
#pragma unroll
                for (int x = 0; x < 4; x++)
                {
                    const int h = x >> 1;
                    z[j][x] *= CODED ? rs[h] * sk[x & 1] : rs[h];
                    if (!all)
                    {
                        const unsigned int key = what.x + j * 8 + 2 * t + (x & 1);
                        if ((what.y >> (j / 2) & 1u) != 0 || !paged_seen(p, v, tok[h], key)) { z[j][x] = -INFINITY; }
                    }
                    float y = z[j][x];
                    if constexpr (CODED) { y += (float)(int)(x & 1 ? ev[j] >> 8 : ev[j] & 255u) - 127.f; }
                    top[h] = fmaxf(top[h], y);
                }
            }
            float c[2] = { 1.f, 1.f };
#pragma unroll
            for (int h = 0; h < 2; h++)
            {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xFFFFFFFFu, top[h], 2));
                if (top[h] > m[h] + 8.f)
                {
                    c[h] = paged_exp2(m[h] - top[h]);    // 0 where nothing came before
                    m[h] = top[h];
                    l[h] *= c[h];
                }
            }
            if (__any_sync(0xFFFFFFFFu, c[0] != 1.f || c[1] != 1.f))
            {
#pragma unroll
                for (int i = 0; i < D / 8; i++)
                {
                    acc[i][0] *= c[0];
                    acc[i][1] *= c[0];
                    acc[i][2] *= c[1];
                    acc[i][3] *= c[1];
                }
            }
            const float base[2] = { m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1] };
#pragma unroll
            for (int sub = 0; sub < S::SUB; sub++)
            {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 2; k++)
                {
                    const int j = sub * 2 + k;
                    float w[4];
#pragma unroll
                    for (int x = 0; x < 4; x++)
                    {
                        w[x] = paged_exp2(z[j][x] - base[x >> 1]);
                        l[x >> 1] += w[x];
                        if constexpr (CODED)
                        {
                            // a byte of a row that is not seen may be anything
                            const float two = paged_two(x & 1 ? ev[j] >> 8 : ev[j] & 255u);
                            w[x] = all || w[x] != 0.f ? w[x] * two : 0.f;
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++)
                    {
                        if constexpr (CODED) { hi[k * 2 + h] = pack_f16x2(w[2 * h], w[2 * h + 1]); }
                        else
                        {
                            const uint32_t u = pack_bf16(w[2 * h], w[2 * h + 1]);
                            hi[k * 2 + h] = u;
                            lo[k * 2 + h] = pack_bf16(w[2 * h] - __uint_as_float(u << 16), w[2 * h + 1] - __uint_as_float(u & 0xFFFF0000u));
                        }
                    }
                }
                // ---- values ----
#pragma unroll
                for (int i = 0; i < S::VI; i++)
                {
                    uint32_t w[4][S::VB / 4];
#pragma unroll
                    for (int h = 0; h < 4; h++)
                    {
                        const uint32_t a = from + UNIT * S::ROW + ((sub * 4 + h) * S::VI + i) * 32 * S::VB - (S::VB == 8 ? lane * 8 : 0);
                        if constexpr (S::VB == 16)
                        {
                            const uint4 x = lds128(a);
                            w[h][0] = x.x, w[h][1] = x.y, w[h][2] = x.z, w[h][3] = x.w;
                        }
                        else
                        {
                            const uint2 x = lds64(a);
                            w[h][0] = x.x, w[h][1] = x.y;
                        }
                    }
#pragma unroll
                    for (int x = 0; x < S::VB / 4; x++)
                    {
                        if constexpr (CODED)
                        {
#pragma unroll
                            for (int y = 0; y < 2; y++)    // the word's elements 2 y and 2 y + 1
                            {
                                const uint32_t a = __byte_perm(w[0][x], w[1][x], y ? 0x7362 : 0x5140), b = __byte_perm(w[2][x], w[3][x], y ? 0x7362 : 0x5140);
                                mma16816<true>(acc[i * S::VE + x * 4 + y * 2], hi, e4m3x2_to_f16x2(a), e4m3x2_to_f16x2(b));
                                mma16816<true>(acc[i * S::VE + x * 4 + y * 2 + 1], hi, e4m3x2_to_f16x2(a >> 16), e4m3x2_to_f16x2(b >> 16));
                            }
                        }
                        else
                        {
#pragma unroll
                            for (int y = 0; y < 2; y++)
                            {
                                const uint32_t a = __byte_perm(w[0][x], w[1][x], y ? 0x7632 : 0x5410), b = __byte_perm(w[2][x], w[3][x], y ? 0x7632 : 0x5410);
                                mma16816<false>(acc[i * S::VE + x * 2 + y], hi, a, b);
                                mma16816<false>(acc[i * S::VE + x * 2 + y], lo, a, b);
                            }
                        }
                    }
                }
            }
            stage = (stage + 1) % RW_STAGES;
        }

        // ---- the warps' parts together, four rows at a time ----
#pragma unroll
        for (int h = 0; h < 2; h++)
        {
            l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
            l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
            if (t == 0)
            {
                max_s[warp][g + 8 * h] = m[h];
                sum_s[warp][g + 8 * h] = l[h];
            }
        }
        const bool whole = cur_s.whole(units);
        const unsigned int VL = paged_ld(p.c.vdim);
        float* piece = p.partial + (2 * (size_t)blockIdx.x + (cur_s.unit == 0 ? 1 : 0)) * paged_piece(RW_ROWS, p.c.vdim);
        const bool vec = paged_vec4<__nv_bfloat16>(p);
        for (unsigned int r0 = 0; r0 < s.rows; r0 += RW_MERGE)
        {
            if (r0 != 0) { __syncthreads(); }
#pragma unroll
            for (int h = 0; h < 2; h++)
            {
                const unsigned int r = g + 8 * h - r0;
                if (r < RW_MERGE)
                {
                    float* to = merge + (warp * RW_MERGE + r) * S::MERGE_LD;
#pragma unroll
                    for (int i = 0; i < S::VI; i++)
                    {
#pragma unroll
                        for (int y = 0; y < 2; y++)
                        {
#pragma unroll
                            for (int x = 0; x < S::VE; x += 4)
                            {
                                store4(to + (i * 8 + 2 * t + y) * S::VE + x, make_float4(acc[i * S::VE + x][2 * h + y], acc[i * S::VE + x + 1][2 * h + y],
                                    acc[i * S::VE + x + 2][2 * h + y], acc[i * S::VE + x + 3][2 * h + y]));
                            }
                        }
                    }
                }
            }
            __syncthreads();
            const unsigned int rows = min(RW_MERGE, s.rows - r0);
            for (unsigned int i = threadIdx.x; i < rows * (VL / 4); i += THREADS)
            {
                const unsigned int r = i / (VL / 4), d = i % (VL / 4) * 4;
                float most = -INFINITY, sum = 0.f;
#pragma unroll
                for (unsigned int x = 0; x < WARPS; x++) { most = fmaxf(most, max_s[x][r0 + r]); }
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (unsigned int x = 0; x < WARPS; x++)
                {
                    const float f = most == -INFINITY ? 1.f : paged_exp2(max_s[x][r0 + r] - most);
                    const float4 y = load4(merge + (x * RW_MERGE + r) * S::MERGE_LD + d);
                    sum = fmaf(f, sum_s[x][r0 + r], sum);
                    o.x = fmaf(f, y.x, o.x);
                    o.y = fmaf(f, y.y, o.y);
                    o.z = fmaf(f, y.z, o.z);
                    o.w = fmaf(f, y.w, o.w);
                }
                if (whole)
                {
                    const unsigned int row = s.r0 + r0 + r, head = kvh * p.G + row % p.G;
                    const float f = paged_factor(p, head, most, sum);
                    if (d < p.c.vdim)
                    {
                        paged_store4((__nv_bfloat16*)p.out + (size_t)(v.start + row / p.G) * p.ldo + (size_t)head * p.c.vdim, d, p.c.vdim, vec,
                            make_float4(o.x * f, o.y * f, o.z * f, o.w * f));
                    }
                }
                else
                {
                    store4(piece + (size_t)(r0 + r) * VL + d, o);
                    if (d == 0)
                    {
                        piece[RW_ROWS * VL + r0 + r] = most;
                        piece[RW_ROWS * VL + RW_ROWS + r0 + r] = sum;
                    }
                }
            }
        }
        if (!whole && cur_s.unit == 0) { header = cur_s.header(share, at, blockIdx.x); }
        at += units;
        __syncthreads();
        if (threadIdx.x == 0 && at < end) { cur_s.next(p); }
    }
    cp_async_wait<0>();
    if (threadIdx.x == 0) { p.header[blockIdx.x] = header; }
}

template <int D, bool CODED>
static int run_rows(PagedParams& p, unsigned int ctas, cudaStream_t stream, bool pdl)
{
    using S = RowsShape<D, CODED>;
    p.least = S::WARPS;    // a unit for every warp
    return launch_kernel("paged_rows", paged_rows_kernel<D, CODED>, dim3(ctas), dim3(32 * S::WARPS), (size_t)S::SMEM, stream, pdl, p);
}

int launch_paged_rows(PagedParams& p, bool coded, unsigned int ctas, cudaStream_t stream, bool pdl)
{
    const unsigned int width = p.c.dim > p.c.vdim ? p.c.dim : p.c.vdim;
    if (coded) { return width <= 64 ? run_rows<64, true>(p, ctas, stream, pdl) : width <= 128 ? run_rows<128, true>(p, ctas, stream, pdl) : run_rows<256, true>(p, ctas, stream, pdl); }
    return width <= 64 ? run_rows<64, false>(p, ctas, stream, pdl) : width <= 128 ? run_rows<128, false>(p, ctas, stream, pdl) : run_rows<256, false>(p, ctas, stream, pdl);
}

}    // namespace b200
