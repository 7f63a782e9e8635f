// Attention of few query rows (up to 16 packed ones per segment: decoding) over a cache in pages, HBM-bound, on mma.sync.
//
// Every warp streams units of its own through a ring in shared memory that only it uses: its first lane asks for the pages' rows by
// TMA, sixteen at a time, and no barrier stands between the warps while they stream.  Both products are turned, so that the few
// queries are the short side of m16n8k16: sixteen keys, then sixteen elements of values, are the rows.  Scores: a lane takes 16 bytes of
// two keys' rows as the k places of several products (the queries' elements are permuted alike).  Values: a lane takes the same
// 16 bytes of four keys; byte permutes pair two keys' elements, two elements make a product's rows.  The weights change their place
// between the two by movmatrix.  Which key is which row is chosen so that, with the 128-byte swizzle, no two lanes of an access
// meet in a bank; for that the lanes of odd rows take a pair of values in the other order.
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

template <int D, bool CODED>
struct RowsShape
{
    static constexpr int EB = CODED ? 1 : 2;
    static constexpr int ROW = D * EB;                                  // bytes of a cache row
    static constexpr int WARPS = ROW > 256 ? 4 : 8;
    static constexpr int STAGES = 3;
    static constexpr int UNIT = ROW >= 256 ? 16 : 4096 / ROW;           // keys: 8 KB a stage (16 KB for the longest rows)
    static constexpr int SUB = UNIT / 16;
    static constexpr int EPC = 16 / EB;                                 // elements of a 16-byte piece
    static constexpr int KI = ROW / 64;                                 // pieces of a key row per lane: i * 4 + lane % 4
    static constexpr int VB = ROW < 128 ? ROW / 8 : 16;                 // bytes of a value piece
    static constexpr int VI = ROW / (8 * VB);                           // pieces of a value row per lane: i * 8 + lane / 4
    static constexpr int VE = VB / EB;                                  // its elements
    static constexpr bool WIDE = ROW >= 128;                            // 128-byte pieces of rows, swizzled; else rows of 64 bytes
    static constexpr int BOX = 16 * (WIDE ? 128 : 64);                  // bytes of one copy
    static constexpr int BOXES = WIDE ? ROW / 128 : 1;                  // copies of sixteen rows
    static constexpr int STAGE = 2 * UNIT * ROW;
    static constexpr int SCALES = CODED ? 2 * UNIT : 0;                 // exponent bytes of a stage
    static constexpr int INFO = 16;                                     // of a stage: first key, subtiles on no page
    static constexpr int MERGE = D > 128 ? 2 : 4;                       // rows that the warps put together at a time
    static constexpr int MERGE_LD = D + 4;
    static constexpr int RING = STAGES * STAGE;
    static constexpr int SMALL = STAGES * (SCALES + INFO);
    static constexpr int SMEM = WARPS * (RING + SMALL) + WARPS * MERGE * MERGE_LD * 4 + 1024;
};

__device__ __forceinline__ uint2 lds64(uint32_t addr)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ unsigned int lds_u8(uint32_t addr)
{
    unsigned int v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
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

// The transpose of an 8 x 8 tile of 16-bit numbers.
__device__ __forceinline__ uint32_t transposed(uint32_t a)
{
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// NT: tiles of eight query rows
template <int D, bool CODED, int NT>
__global__ void __launch_bounds__(32 * RowsShape<D, CODED>::WARPS, 1) paged_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
    const __grid_constant__ PagedParams p, unsigned int* status)
{
    using S = RowsShape<D, CODED>;
    constexpr unsigned int UNIT = S::UNIT, MERGE = S::MERGE, WARPS = S::WARPS, THREADS = 32 * WARPS, ROWS = 8 * NT;
    constexpr int STEPS = D / 16;
    extern __shared__ unsigned char rw_raw[];
    unsigned char* rw_smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(rw_raw) + 1023) & ~(uintptr_t)1023);
    __shared__ uint64_t full[WARPS][S::STAGES];
    __shared__ PagedShare share;
    __shared__ unsigned long long sums[WARPS];
    __shared__ PagedCursor<UNIT, ROWS> cur_s;
    __shared__ float max_s[WARPS][ROWS], sum_s[WARPS][ROWS];
    const unsigned int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    unsigned char* ring = rw_smem + warp * S::RING;
    unsigned char* small = rw_smem + WARPS * S::RING + warp * S::SMALL;    // per stage: info, exponents of keys, of values
    float* merge = reinterpret_cast<float*>(rw_smem + WARPS * (S::RING + S::SMALL));

    if (threadIdx.x == 0)
    {
        for (unsigned int i = 0; i < WARPS * S::STAGES; i++) { mbar_init(&full[0][0] + i, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    grid_dependency_launch();
    grid_dependency_wait();
    paged_share<UNIT, ROWS, THREADS>(p, sums, &share);
    if (share.begin >= share.end)
    {
        if (threadIdx.x == 0) { p.header[blockIdx.x] = PagedHeader{}; }
        return;
    }
    const unsigned int end = (unsigned int)(share.end - share.begin);    // places are counted from the share's first unit on

    // ---- what the warp asks for: units warp, warp + WARPS, ... of the share, across its segments ----
    PagedCursor<UNIT, ROWS> ask;
    unsigned int ask_at = warp, ask_seg = 0;    // the unit, and where its segment's units in the share begin
    ask.at(p, share);
    unsigned int ask_key = 0;
    int ask_page = -1;    // lane i: the page of the unit's i-th sixteen keys as the table has it; looked at only when it is needed, a unit later
    auto find = [&]() {
        if (ask_at >= end) { return; }
        for (unsigned int n = ask.s.count - ask.unit; ask_at - ask_seg >= n; n = ask.s.count)
        {
            ask_seg += n;
            ask.next(p);
        }
        ask_key = ask.s.unit(ask.unit + (ask_at - ask_seg)) * UNIT;
        const unsigned int first = ask_key + lane * 16;
        ask_page = -1;
        // a range of keys meets one of the two wanted ranges
        if (lane < (unsigned int)S::SUB && first < ask.s.lim && (first + 16 > ask.s.low || (first + 16 > ask.v.floor && first < ask.s.first_end)))
        {
            const unsigned int i = first >> p.c.shift;    // (lim is 0 for a slot that is none, and nowhere behind the table's row)
            ask_page = p.c.table[(size_t)(unsigned int)ask.v.slot * p.c.ld_table + i];
        }
    };
    unsigned int asked = 0;    // units
    auto request = [&]() {
        if (ask_at >= end) { return; }
        const unsigned int stage = asked % S::STAGES;
        unsigned char* to = ring + stage * S::STAGE;
        unsigned char* info = small + stage * (S::INFO + S::SCALES);
        const bool none = (unsigned int)ask_page >= p.c.pages;
        const unsigned int bad = __ballot_sync(0xFFFFFFFFu, lane < (unsigned int)S::SUB && none);
        if (none) { ask_page = (int)p.c.pages; }    // behind the caches' end: zeros
        if (lane == 0)
        {
            *reinterpret_cast<uint2*>(info) = make_uint2(ask_key, bad);
            mbar_expect_tx(&full[warp][stage], S::STAGE + (CODED ? 32 * (S::SUB - __popc(bad)) : 0));
        }
        __syncwarp();
        // lane i asks for the i-th sixteen keys
        if (lane < (unsigned int)S::SUB)
        {
            const unsigned int at = (ask.kvh << p.c.shift) + ((ask_key + lane * 16) & ((1u << p.c.shift) - 1u));
#pragma unroll
            for (int i = 0; i < S::BOXES; i++)
            {
                tma_load_3d(to + (lane * S::BOXES + i) * S::BOX, &tmK, i * (128 / S::EB), (int)at, ask_page, &full[warp][stage]);
                tma_load_3d(to + UNIT * S::ROW + (lane * S::BOXES + i) * S::BOX, &tmV, i * (128 / S::EB), (int)at, ask_page, &full[warp][stage]);
            }
            if (CODED && !none)
            {
                const size_t from = ((size_t)(unsigned int)ask_page * p.c.Hkv << p.c.shift) + at;
                bulk_g2s(info + S::INFO + lane * 16, p.c.k_scale + from, 16, &full[warp][stage]);
                bulk_g2s(info + S::INFO + UNIT + lane * 16, p.c.v_scale + from, 16, &full[warp][stage]);
            }
        }
        __syncwarp();
        if (lane == 0) { mbar_arrive(&full[warp][stage]); }
        asked++;
        ask_at += WARPS;
        find();
    };
    find();
#pragma unroll
    for (int s = 0; s + 1 < S::STAGES; s++) { request(); }
    unsigned int taken = 0;    // units
    bool lost = false;         // a wait has run out: nothing more is taken
    // Rows of the products: key `order(i)` of eight is row i.  Where a lane finds its pieces of a copy.
    auto order = [](unsigned int i) { return (i >> 1) ^ ((i & 1u) * (S::WIDE ? 4u : 5u)); };
    const unsigned int key_g = order(g);
    const uint32_t k_at = S::WIDE ? key_g * 128 + ((t ^ key_g) << 4) : key_g * 64 + t * 16;
    const unsigned int swap = S::WIDE ? g & 1u : 0u;    // in which order a pair of values is taken
    uint32_t v_at[2];
#pragma unroll
    for (unsigned int x = 0; x < 2; x++)
    {
        const unsigned int r = order(2 * t + (x ^ swap));
        v_at[x] = S::WIDE ? r * 128 + ((g ^ r) << 4) : r * 64 + g * 8;
    }
    const uint32_t pair[2] = { CODED ? (swap ? 0x1504u : 0x5140u) : (swap ? 0x1054u : 0x5410u), CODED ? (swap ? 0x3726u : 0x7362u) : (swap ? 0x3276u : 0x7632u) };

    if (threadIdx.x == 0) { cur_s.at(p, share); }
    PagedHeader header = {};
    unsigned int at = 0, mine = warp;    // the segment's first unit; the warp's next unit
    while (at < end)
    {
        __syncthreads();
        const PagedEntry v = cur_s.v;
        const PagedSegment s = cur_s.s;
        const unsigned int kvh = cur_s.kvh, units = cur_s.take(end - at);
        // ---- queries: row g of each tile as an operand; the scores' columns are the rows 2 t and 2 t + 1 ----
        uint32_t q[NT][STEPS][2];
        float rs[NT][2];
        unsigned int tok[NT][2];    // those rows' tokens' positions
#pragma unroll
        for (int n = 0; n < NT; n++)
        {
            const unsigned int r = s.r0 + n * 8 + g;
            const bool real = n * 8 + g < s.rows;
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
                q[n][k][0] = u.x;
                q[n][k][1] = u.y;
                if constexpr (CODED)
                {
                    top = max(max(top, max((u.x << 16) & 0x7FFF0000u, u.x & 0x7FFF0000u)), max((u.y << 16) & 0x7FFF0000u, u.y & 0x7FFF0000u));
                }
            }
            float scale = p.scale * 1.44269504088896341f;
            if constexpr (CODED)
            {
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                // the largest element comes to 2^14 .. 2^15
                const unsigned int b = min(268u - (top >> 23), 254u);
                const float f = paged_two(b);
                scale *= b == 254u ? 5.877471754e-39f : paged_two(254u - b);    // 2^-127 is not a normal number
#pragma unroll
                for (int k = 0; k < STEPS; k++)
                {
#pragma unroll
                    for (int x = 0; x < 2; x++)
                    {
                        q[n][k][x] = pack_f16x2(__uint_as_float(q[n][k][x] << 16) * f, __uint_as_float(q[n][k][x] & 0xFFFF0000u) * f);
                    }
                }
            }
#pragma unroll
            for (unsigned int x = 0; x < 2; x++)
            {
                rs[n][x] = __shfl_sync(0xFFFFFFFFu, scale, 8 * t + 4 * x);    // of the lane that holds row 2 t + x
                const unsigned int i = n * 8 + 2 * t + x;
                tok[n][x] = v.pos + (i < s.rows ? (s.r0 + i) / p.G : 0);
            }
        }
        float acc[D / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
        {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < D / 16; i++) { acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.f; }
        }
        // keys that every row sees
        const unsigned int lim_all = min(v.pos + s.r0 / p.G + 1, s.lim), t_last = v.pos + (s.r0 + s.rows - 1) / p.G;
        const unsigned int low_all = max(v.floor, p.window != 0 && t_last + 1 > p.window ? t_last + 1 - p.window : 0u);

        for (; mine < at + units; mine += WARPS)
        {
            const unsigned int stage = taken % S::STAGES;
            if (!__all_sync(0xFFFFFFFFu, !lost && mbar_wait_bounded(&full[warp][stage], (taken / S::STAGES) & 1u)))
            {
                if (!lost && lane == 0) { note_timeout(status, WAIT_PAGED_ROWS, warp & 15u, taken); }
                lost = true;
                break;
            }
            request();    // into the place of the unit before this one, which every lane is done with
            const uint32_t from = smem_u32(ring) + stage * S::STAGE, from_v = from + UNIT * S::ROW;
            const uint32_t info = smem_u32(small) + stage * (S::INFO + S::SCALES);
            const uint2 what = lds64(info);
            // ---- scores: z[sub][tile][keys g, g + 8][rows 2 t, 2 t + 1] ----
            float z[S::SUB][NT][4];
#pragma unroll
            for (int sub = 0; sub < S::SUB; sub++)
            {
#pragma unroll
                for (int n = 0; n < NT; n++) { z[sub][n][0] = z[sub][n][1] = z[sub][n][2] = z[sub][n][3] = 0.f; }
            }
#pragma unroll
            for (int i = 0; i < S::KI; i++)
            {
#pragma unroll
                for (int sub = 0; sub < S::SUB; sub++)
                {
                    const uint4 x = lds128(from + (sub * S::BOXES + i / 2) * S::BOX + (k_at ^ (i % 2 * 64))),
                                y = lds128(from + (sub * S::BOXES + i / 2) * S::BOX + 8 * (S::BOX / 16) + (k_at ^ (i % 2 * 64)));
                    const uint32_t w[2][4] = { { x.x, x.y, x.z, x.w }, { y.x, y.y, y.z, y.w } };
                    if constexpr (CODED)
                    {
#pragma unroll
                        for (int c = 0; c < 4; c++)
                        {
                            uint32_t a[4];
                            e4m3x4_to_f16x2(w[0][c], a[0], a[2]);
                            e4m3x4_to_f16x2(w[1][c], a[1], a[3]);
#pragma unroll
                            for (int n = 0; n < NT; n++) { mma16816<true>(z[sub][n], a, q[n][i * 4 + c][0], q[n][i * 4 + c][1]); }
                        }
                    }
                    else
                    {
#pragma unroll
                        for (int c = 0; c < 2; c++)
                        {
                            const uint32_t a[4] = { w[0][2 * c], w[1][2 * c], w[0][2 * c + 1], w[1][2 * c + 1] };
#pragma unroll
                            for (int n = 0; n < NT; n++) { mma16816<false>(z[sub][n], a, q[n][i * 2 + c][0], q[n][i * 2 + c][1]); }
                        }
                    }
                }
            }
            // ---- weights ----
            float top[NT][2], sv[S::SUB][2];
#pragma unroll
            for (int n = 0; n < NT; n++) { top[n][0] = top[n][1] = -INFINITY; }
            const bool all = what.y == 0 && what.x >= low_all && what.x + UNIT <= lim_all;
            float u[S::SUB][2];    // log2 of the values' powers of two
#pragma unroll
            for (int sub = 0; sub < S::SUB; sub++)
            {
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    float sk = 1.f;
                    u[sub][h] = 0.f;
                    if constexpr (CODED)
                    {
                        sk = paged_two(lds_u8(info + S::INFO + sub * 16 + h * 8 + key_g));
                        // (a byte of a row that is not seen may be anything: 255 would be no number)
                        const unsigned int b = min(lds_u8(info + S::INFO + UNIT + sub * 16 + h * 8 + key_g), 254u);
                        u[sub][h] = (float)(int)(b - 127u);
                        sv[sub][h] = paged_two(b);
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
                    {
#pragma unroll
                        for (int x = 0; x < 2; x++) { z[sub][n][2 * h + x] *= CODED ? rs[n][x] * sk : rs[n][x]; }
                    }
                }
            }
            if (!all)
            {
#pragma unroll
                for (int sub = 0; sub < S::SUB; sub++)
                {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                    {
                        const unsigned int key = what.x + sub * 16 + h * 8 + key_g;
#pragma unroll
                        for (int n = 0; n < NT; n++)
                        {
#pragma unroll
                            for (int x = 0; x < 2; x++)
                            {
                                if ((what.y >> sub & 1u) != 0 || !paged_seen(p, v, tok[n][x], key)) { z[sub][n][2 * h + x] = -INFINITY; }
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int sub = 0; sub < S::SUB; sub++)
            {
#pragma unroll
                for (int n = 0; n < NT; n++)
                {
#pragma unroll
                    for (int x = 0; x < 2; x++) { top[n][x] = fmaxf(top[n][x], fmaxf(z[sub][n][x] + u[sub][0], z[sub][n][2 + x] + u[sub][1])); }
                }
            }
            // (the maximum is the same in all lanes of a column: most units end with the vote)
            bool grown = false;
#pragma unroll
            for (int n = 0; n < NT; n++) { grown = grown || top[n][0] > m[n][0] + 8.f || top[n][1] > m[n][1] + 8.f; }
            if (__any_sync(0xFFFFFFFFu, grown))
            {
                float c[NT][2];
#pragma unroll
                for (int n = 0; n < NT; n++)
                {
#pragma unroll
                    for (int x = 0; x < 2; x++)
                    {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) { top[n][x] = fmaxf(top[n][x], __shfl_xor_sync(0xFFFFFFFFu, top[n][x], o)); }
                        c[n][x] = 1.f;
                        if (top[n][x] > m[n][x] + 8.f)
                        {
                            c[n][x] = paged_exp2(m[n][x] - top[n][x]);    // 0 where nothing came before
                            m[n][x] = top[n][x];
                            l[n][x] *= c[n][x];
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < D / 16; i++)
                {
#pragma unroll
                    for (int n = 0; n < NT; n++)
                    {
                        acc[i][n][0] *= c[n][0];
                        acc[i][n][1] *= c[n][1];
                        acc[i][n][2] *= c[n][0];
                        acc[i][n][3] *= c[n][1];
                    }
                }
            }
            uint32_t hi[S::SUB][NT][2], lo[S::SUB][NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++)
            {
                const float base[2] = { m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1] };
#pragma unroll
                for (int sub = 0; sub < S::SUB; sub++)
                {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                    {
                        float w[2];
#pragma unroll
                        for (int x = 0; x < 2; x++)
                        {
                            w[x] = paged_exp2(z[sub][n][2 * h + x] - base[x]);
                            l[n][x] += w[x];
                            if constexpr (CODED) { w[x] *= sv[sub][h]; }
                        }
                        if constexpr (CODED) { hi[sub][n][h] = transposed(pack_f16x2(w[0], w[1])); }
                        else
                        {
                            const uint32_t a = pack_bf16(w[0], w[1]);
                            hi[sub][n][h] = transposed(a);
                            lo[sub][n][h] = transposed(pack_bf16(w[0] - __uint_as_float(a << 16), w[1] - __uint_as_float(a & 0xFFFF0000u)));
                        }
                    }
                }
            }
            // ---- values ----
#pragma unroll
            for (int sub = 0; sub < S::SUB; sub++)
            {
#pragma unroll
                for (int i = 0; i < S::VI; i++)
                {
                    uint32_t w[4][S::VB / 4];
#pragma unroll
                    for (int h = 0; h < 4; h++)
                    {
                        const uint32_t at = from_v + (sub * S::BOXES + i) * S::BOX + (h >> 1) * 8 * (S::BOX / 16) + v_at[h & 1];
                        if constexpr (S::VB == 16)
                        {
                            const uint4 x = lds128(at);
                            w[h][0] = x.x, w[h][1] = x.y, w[h][2] = x.z, w[h][3] = x.w;
                        }
                        else
                        {
                            const uint2 x = lds64(at);
                            w[h][0] = x.x, w[h][1] = x.y;
                        }
                        if (!all && !paged_wanted(v, s, what.x + sub * 16 + (h >> 1) * 8 + order(2 * t + ((h & 1) ^ swap))))
                        {
#pragma unroll
                            for (int x = 0; x < S::VB / 4; x++) { w[h][x] = 0; }    // nobody's: it may be no number, and 0 times that none either
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
                                uint32_t a[4];
                                e4m3x4_to_f16x2(__byte_perm(w[0][x], w[1][x], pair[y]), a[0], a[1]);
                                e4m3x4_to_f16x2(__byte_perm(w[2][x], w[3][x], pair[y]), a[2], a[3]);
#pragma unroll
                                for (int n = 0; n < NT; n++) { mma16816<true>(acc[i * S::VE / 2 + x * 2 + y][n], a, hi[sub][n][0], hi[sub][n][1]); }
                            }
                        }
                        else
                        {
                            const uint32_t a[4] = { __byte_perm(w[0][x], w[1][x], pair[0]), __byte_perm(w[0][x], w[1][x], pair[1]), __byte_perm(w[2][x], w[3][x], pair[0]),
                                __byte_perm(w[2][x], w[3][x], pair[1]) };
#pragma unroll
                            for (int n = 0; n < NT; n++)
                            {
                                mma16816<false>(acc[i * S::VE / 2 + x][n], a, hi[sub][n][0], hi[sub][n][1]);
                                mma16816<false>(acc[i * S::VE / 2 + x][n], a, lo[sub][n][0], lo[sub][n][1]);
                            }
                        }
                    }
                }
            }
            taken++;
            __syncwarp();
        }

        // ---- the warps' parts together, a few rows at a time ----
#pragma unroll
        for (int n = 0; n < NT; n++)
        {
#pragma unroll
            for (int x = 0; x < 2; x++)
            {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) { l[n][x] += __shfl_xor_sync(0xFFFFFFFFu, l[n][x], o); }
                if (g == 0)
                {
                    max_s[warp][n * 8 + 2 * t + x] = m[n][x];
                    sum_s[warp][n * 8 + 2 * t + x] = l[n][x];
                }
            }
        }
        const bool whole = cur_s.whole(units);
        const unsigned int VL = paged_ld(p.c.vdim);
        float* piece = p.partial + (2 * (size_t)blockIdx.x + (cur_s.unit == 0 ? 1 : 0)) * paged_piece(ROWS, p.c.vdim);
        const bool vec = paged_vec4<__nv_bfloat16>(p);
        for (unsigned int r0 = 0; r0 < s.rows; r0 += MERGE)
        {
            if (r0 != 0) { __syncthreads(); }
#pragma unroll
            for (int n = 0; n < NT; n++)
            {
#pragma unroll
                for (int y = 0; y < 2; y++)
                {
                    const unsigned int r = n * 8 + 2 * t + y - r0;
                    if (r < MERGE)
                    {
                        float* to = merge + (warp * MERGE + r) * S::MERGE_LD;
#pragma unroll
                        for (int i = 0; i < S::VI; i++)
                        {
#pragma unroll
                            for (int x = 0; x < S::VE / 2; x += 2)
                            {
                                const int k = i * S::VE / 2 + x;
                                store4(to + (i * 8 + g) * S::VE + 2 * x, make_float4(acc[k][n][y], acc[k][n][2 + y], acc[k + 1][n][y], acc[k + 1][n][2 + y]));
                            }
                        }
                    }
                }
            }
            __syncthreads();
            const unsigned int rows = min(MERGE, s.rows - r0);
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
                    const float4 y = load4(merge + (x * MERGE + r) * S::MERGE_LD + d);
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
                        piece[ROWS * VL + r0 + r] = most;
                        piece[ROWS * VL + ROWS + r0 + r] = sum;
                    }
                }
            }
        }
        if (!whole && cur_s.unit == 0) { header = cur_s.header(share, share.begin + at, blockIdx.x); }
        at += units;
        __syncthreads();
        if (threadIdx.x == 0 && at < end) { cur_s.next(p); }
    }
    if (lost && lane == 0)
    {
        // wait (bounded) for the copies in flight before the CTA may leave
        for (; taken < asked; taken++) { mbar_wait_bounded(&full[warp][taken % S::STAGES], (taken / S::STAGES) & 1u); }
    }
    if (threadIdx.x == 0) { p.header[blockIdx.x] = header; }
}

template <int D, bool CODED>
static int run_rows(PagedParams& p, unsigned int rows, unsigned int ctas, cudaStream_t stream, bool pdl)
{
    using S = RowsShape<D, CODED>;
    p.least = S::WARPS;    // a unit for every warp
    const dim3 grid(ctas), block(32 * S::WARPS);
    unsigned int* status = decoder_status_word();
    if (!status) { return 1; }
    CUtensorMap tk, tv;
    const unsigned int cols = (S::WIDE ? 128 : 64) / S::EB;
    if (!make_paged_map(&tk, CODED, p.c.k, p.c.k_ld, p.c, cols, 16, S::WIDE) || !make_paged_map(&tv, CODED, p.c.v, p.c.v_ld, p.c, cols, 16, S::WIDE)) { return -1; }
    return rows <= 8 ? launch_kernel("paged_rows", paged_rows_kernel<D, CODED, 1>, grid, block, (size_t)S::SMEM, stream, pdl, tk, tv, p, status)
                     : launch_kernel("paged_rows", paged_rows_kernel<D, CODED, 2>, grid, block, (size_t)S::SMEM, stream, pdl, tk, tv, p, status);
}

int launch_paged_rows(PagedParams& p, bool coded, unsigned int rows, unsigned int ctas, cudaStream_t stream, bool pdl)
{
    const unsigned int width = p.c.dim > p.c.vdim ? p.c.dim : p.c.vdim;
    if (coded)
    {
        return width <= 64 ? run_rows<64, true>(p, rows, ctas, stream, pdl) : width <= 128 ? run_rows<128, true>(p, rows, ctas, stream, pdl)
                                                                                           : run_rows<256, true>(p, rows, ctas, stream, pdl);
    }
    return width <= 64 ? run_rows<64, false>(p, rows, ctas, stream, pdl) : width <= 128 ? run_rows<128, false>(p, rows, ctas, stream, pdl)
                                                                                        : run_rows<256, false>(p, rows, ctas, stream, pdl);
}

}    // namespace b200
