// How a ragged batch over a cache in pages is dealt out to workers (CTAs, or their warps), and which keys its rows see.  Nothing here needs a GPU, so that it can
// be looked at without one.
//
// A segment is a kv head of an entry with up to ROWS packed query rows (tokens x heads of the kv head); its keys come in units of
// UNIT, those of the window and, with a window, those of the first keys.  All segments' units lie one behind the other, entry by
// entry, and every worker takes an equal share of them: long and short sequences, one sequence or many come out even, and no
// length has to be known on the host.  A share's segments that are whole are written out; of the (at most two) others the worker
// leaves maximum, sum and weighted values in the scratch, and a second kernel puts the pieces together in their order, so that the
// same call gives the same bits.
#pragma once

#include <cstddef>

#if defined(__CUDACC__)
#define B200_PLAN __host__ __device__ __forceinline__
#else
#define B200_PLAN inline
#endif

namespace b200
{

template <class T>
B200_PLAN T plan_min(T a, T b)
{
    return a < b ? a : b;
}
template <class T>
B200_PLAN T plan_max(T a, T b)
{
    return a < b ? b : a;
}

// a / b; the short division where it will do (a long one takes the GPU a hundred instructions)
B200_PLAN unsigned long long plan_div(unsigned long long a, unsigned long long b)
{
    return ((a | b) >> 32) == 0 ? (unsigned int)a / (unsigned int)b : a / b;
}

struct PagedCache
{
    unsigned char *k, *v, *k_scale, *v_scale;
    const int* table;
    unsigned int pages, shift, slots, ld_table, Hkv, dim, vdim, k_ld, v_ld;    // 1 << shift rows a page
    unsigned int cap;                                                          // positions a table row covers
};

struct PagedBatch
{
    const int *slot, *pos, *start, *n, *token_entry, *floor;
    unsigned int e0, entries, t0, tokens, max_n;
};

// What the dealing out goes by.
struct PagedPlan
{
    PagedCache c;
    PagedBatch b;
    unsigned int G, window, first;    // query heads per kv head
    unsigned int least;               // units a worker gets at least, where there are enough
};

// The segment that a CTA leaves unfinished.
struct PagedHeader
{
    unsigned int pieces;            // its own and those of the CTAs behind it; 0: there is no such segment
    unsigned int worker;            // that has begun it
    unsigned int rows, r0;          // packed query rows, the first one
    unsigned int start, kvh;        // the entry's first token
};

// The page of a sequence's position, or -1.
B200_PLAN int paged_page(const PagedCache& c, int slot, unsigned int at)
{
    const unsigned int i = at >> c.shift;
    if (slot < 0 || i >= c.ld_table) { return -1; }
    const int page = c.table[(size_t)slot * c.ld_table + i];
    return (unsigned int)page < c.pages ? page : -1;
}
// Row of the caches (and of their scales) that holds a kv head's key at `at`.
B200_PLAN size_t paged_row(const PagedCache& c, int page, unsigned int kvh, unsigned int at)
{
    return (((size_t)page * c.Hkv + kvh) << c.shift) + (at & ((1u << c.shift) - 1u));
}
// An entry as the kernels take it: tokens outside the call's, a negative position or length, a slot that is none are left out.
struct PagedEntry
{
    unsigned int pos, n, start, floor;
    int slot;
};
B200_PLAN PagedEntry paged_entry(const PagedPlan& p, unsigned int e)
{
    const int n = p.b.n[e], pos = p.b.pos[e], start = p.b.start[e], slot = p.b.slot[e];
    const int floor = p.b.floor != nullptr ? p.b.floor[e] : 0;
    PagedEntry v;
    const unsigned int at = (unsigned int)start - p.b.t0;
    v.n = n > 0 && pos >= 0 && start >= 0 && (unsigned int)start >= p.b.t0 && at < p.b.tokens ? plan_min(plan_min((unsigned int)n, p.b.max_n), p.b.tokens - at) : 0u;
    v.pos = (unsigned int)pos;
    v.start = (unsigned int)start;
    v.floor = floor > 0 ? (unsigned int)floor : 0u;
    v.slot = (unsigned int)slot < p.c.slots ? slot : -1;
    return v;
}

// The keys that some row of a segment sees: floor .. first_end - 1 and low .. lim - 1, and the units that hold them.
struct PagedSegment
{
    unsigned int r0, rows;                  // its packed rows
    unsigned int first_end, low, lim;
    unsigned int a0, a, b0, count;          // units a0 .. a0 + a - 1, then b0 ..; `count` in all, at least 1
    B200_PLAN unsigned int unit(unsigned int i) const { return i < a ? a0 + i : b0 + (i - a); }
};
template <unsigned int UNIT, unsigned int ROWS>
B200_PLAN PagedSegment paged_segment(const PagedPlan& p, const PagedEntry& v, unsigned int rt)
{
    PagedSegment s;
    s.r0 = rt * ROWS;
    s.rows = plan_min(ROWS, v.n * p.G - s.r0);
    const unsigned int t0 = v.pos + s.r0 / p.G, t1 = v.pos + (s.r0 + s.rows - 1) / p.G;
    s.lim = v.slot < 0 ? 0u : plan_min(t1 + 1, p.c.cap);
    s.low = plan_max(v.floor, p.window != 0 && t0 + 1 > p.window ? t0 + 1 - p.window : 0u);
    s.first_end = v.floor;
    if (p.window != 0 && v.floor < s.lim) { s.first_end = v.floor + plan_min(p.first, s.lim - v.floor); }
    s.a0 = v.floor / UNIT;
    s.a = s.first_end > v.floor ? (s.first_end + UNIT - 1) / UNIT - s.a0 : 0u;
    s.b0 = s.low / UNIT;
    if (s.a != 0) { s.b0 = plan_max(s.b0, s.a0 + s.a); }
    const unsigned int end = (s.lim + UNIT - 1) / UNIT;
    s.count = plan_max(1u, s.a + (s.lim > s.low && end > s.b0 ? end - s.b0 : 0u));
    return s;
}
template <unsigned int ROWS>
B200_PLAN unsigned int paged_tiles(const PagedPlan& p, const PagedEntry& v)
{
    return (v.n * p.G + ROWS - 1) / ROWS;
}
// Does some row of the segment see the key?  Does the row of the token at t?
B200_PLAN bool paged_wanted(const PagedEntry& v, const PagedSegment& s, unsigned int key)
{
    return key < s.lim && (key >= s.low || (key >= v.floor && key < s.first_end));
}
B200_PLAN bool paged_seen(const PagedPlan& p, const PagedEntry& v, unsigned int t, unsigned int key)
{
    return key >= v.floor && key <= t && key < p.c.cap && (p.window == 0 || t - key < p.window || key - v.floor < p.first);
}

// A worker's share.
struct PagedShare
{
    unsigned long long total, begin, end;
    unsigned int workers;            // that have a share
    unsigned int e, kvh, rt, unit;   // where `begin` lies
};
// Workers that get a share, and where the share of worker w begins.
B200_PLAN unsigned int paged_workers(unsigned long long total, unsigned int least, unsigned int most)
{
    const unsigned long long fit = plan_div(total, least);
    return fit == 0 ? 1u : fit < most ? (unsigned int)fit : most;
}
B200_PLAN unsigned long long paged_begin(unsigned long long total, unsigned int w, unsigned int workers) { return w < workers ? plan_div(total * w, workers) : total; }

// Units of one head of an entry.
template <unsigned int UNIT, unsigned int ROWS>
B200_PLAN unsigned long long paged_head_units(const PagedPlan& p, const PagedEntry& v)
{
    unsigned long long sum = 0;
    const unsigned int tiles = paged_tiles<ROWS>(p, v);
    for (unsigned int rt = 0; rt < tiles; rt++) { sum += paged_segment<UNIT, ROWS>(p, v, rt).count; }
    return sum;
}
// The segment and unit at `at`, counted from entry e's first unit on.
template <unsigned int UNIT, unsigned int ROWS>
B200_PLAN void paged_find(const PagedPlan& p, unsigned int e, unsigned int e_end, unsigned long long at, PagedShare* share)
{
    for (; e < e_end; e++)
    {
        const PagedEntry v = paged_entry(p, e);
        const unsigned long long head = paged_head_units<UNIT, ROWS>(p, v);
        if (at >= head * p.c.Hkv)
        {
            at -= head * p.c.Hkv;
            continue;
        }
        share->e = e;
        share->kvh = (unsigned int)plan_div(at, head);
        at -= share->kvh * head;
        unsigned int rt = 0;
        for (unsigned int n = paged_segment<UNIT, ROWS>(p, v, 0).count; at >= n; n = paged_segment<UNIT, ROWS>(p, v, ++rt).count) { at -= n; }
        share->rt = rt;
        share->unit = (unsigned int)at;
        return;
    }
}

// Walks a share's segments.
template <unsigned int UNIT, unsigned int ROWS>
struct PagedCursor
{
    unsigned int e, kvh, rt, unit;    // the segment, and its first unit in the share
    PagedEntry v;
    PagedSegment s;
    B200_PLAN void at(const PagedPlan& p, const PagedShare& share)
    {
        e = share.e;
        kvh = share.kvh;
        rt = share.rt;
        unit = share.unit;
        v = paged_entry(p, e);
        s = paged_segment<UNIT, ROWS>(p, v, rt);
    }
    // There is a next segment.
    B200_PLAN void next(const PagedPlan& p)
    {
        unit = 0;
        if (++rt >= paged_tiles<ROWS>(p, v))
        {
            rt = 0;
            if (++kvh >= p.c.Hkv)
            {
                kvh = 0;
                do
                {
                    e++;
                    v = paged_entry(p, e);
                } while (v.n == 0 && e + 1 < p.b.e0 + p.b.entries);
            }
        }
        s = paged_segment<UNIT, ROWS>(p, v, rt);
    }
    // Units of the segment in a share of which `left` units are left, and whether that is all of them.
    B200_PLAN unsigned int take(unsigned long long left) const { return (unsigned int)plan_min((unsigned long long)(s.count - unit), left); }
    B200_PLAN bool whole(unsigned int taken) const { return taken == s.count; }
    // The worker whose share holds the segment's last unit, where `begin` is the global unit of the first one in the share.
    B200_PLAN unsigned int last(const PagedShare& share, unsigned long long begin) const
    {
        return (unsigned int)plan_div((begin + (s.count - unit)) * share.workers - 1, share.total);
    }
};

}    // namespace b200
