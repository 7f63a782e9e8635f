"""How a ragged batch over a paged cache is dealt out to workers, and what the calls refuse.  No GPU needed: the rules are host code, and
a refused call launches nothing."""
import ctypes as C
import subprocess

import numpy as np
import pytest

from __graft_entry__ import ROOT, load_package

SHAPES = [(32, 4), (32, 16), (16, 16), (64, 16), (128, 128), (128, 256)]    # keys per unit, rows per segment


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    top = tmp_path_factory.mktemp("plan")
    (top / "plan.cpp").write_text('''
#include "%s/cccc-lite_b200/csrc/decoder/paged_plan.cuh"
using namespace b200;
// Walks every worker's share.  hits[e][kvh][token][key]: times a row that sees the key meets it (the first head of the token); taken[e][kvh][key]:
// the key's row is fetched.  Returns the number of rules that were broken.
template <unsigned U, unsigned R>
static int walk(const PagedPlan& p, unsigned grid, unsigned max_t, unsigned max_k, int* hits, int* fetched, int* pieces)
{
    int bad = 0;
    unsigned long long total = 0;
    for (unsigned e = p.b.e0; e < p.b.e0 + p.b.entries; e++) { total += paged_head_units<U, R>(p, paged_entry(p, e)) * p.c.Hkv; }
    const unsigned ctas = paged_workers(total, p.least, grid);
    unsigned expect = 0;    // pieces of an unfinished segment still to come
    struct { unsigned e, kvh, rt, last; } open = {};
    for (unsigned c = 0; c < grid; c++)
    {
        PagedShare s = {};
        s.total = total, s.workers = ctas, s.begin = paged_begin(total, c, ctas), s.end = paged_begin(total, c + 1, ctas);
        if (c >= ctas && s.begin != s.end) { bad++; }
        if (s.begin >= s.end) { continue; }
        if (s.end - s.begin > (total + ctas - 1) / ctas || (total / p.least >= 1 && s.end - s.begin < p.least)) { bad++; }
        paged_find<U, R>(p, p.b.e0, p.b.e0 + p.b.entries, s.begin, &s);
        PagedCursor<U, R> cur;
        cur.at(p, s);
        bool first = true;
        for (unsigned long long at = s.begin; at < s.end; first = false)
        {
            const unsigned units = cur.take(s.end - at);
            if (units == 0 || cur.v.n == 0 || cur.e >= p.b.e0 + p.b.entries) { return bad + 1000; }
            const bool whole = cur.whole(units);
            if (cur.unit != 0)    // a piece of the segment that a worker before left open
            {
                if (!first || expect == 0 || open.e != cur.e || open.kvh != cur.kvh || open.rt != cur.rt || cur.last(s, at) != open.last) { bad++; }
                expect--;
                if ((cur.unit + units == cur.s.count) != (expect == 0)) { bad++; }
            }
            else if (!whole)
            {
                if (expect != 0) { bad++; }
                open = { cur.e, cur.kvh, cur.rt, cur.last(s, at) };
                expect = open.last - c;
                if (at + units != s.end || open.last <= c || open.last >= ctas) { bad++; }
                pieces[0]++;
            }
            for (unsigned u = 0; u < units; u++)
            {
                for (unsigned k = 0; k < U; k++)
                {
                    const unsigned key = cur.s.unit(cur.unit + u) * U + k;
                    if (!paged_wanted(cur.v, cur.s, key)) { continue; }
                    if (key >= max_k || paged_page(p.c, cur.v.slot, key) < -1) { return bad + 100; }
                    fetched[((cur.e * p.c.Hkv) + cur.kvh) * max_k + key]++;
                    for (unsigned r = 0; r < cur.s.rows; r++)
                    {
                        const unsigned row = cur.s.r0 + r, t = row / p.G;
                        if (row %% p.G == 0 && paged_seen(p, cur.v, cur.v.pos + t, key)) { hits[(((size_t)cur.e * p.c.Hkv + cur.kvh) * max_t + t) * max_k + key]++; }
                    }
                }
            }
            at += units;
            if (at < s.end) { cur.next(p); }
        }
    }
    return bad + (expect != 0);
}
extern "C" int run(int shape, const int* slot, const int* pos, const int* start, const int* n, const int* floor, unsigned entries, unsigned e0, unsigned tokens,
    unsigned t0, unsigned max_n, unsigned slots, unsigned cap, unsigned Hkv, unsigned G, unsigned window, unsigned first, unsigned least, unsigned grid,
    const int* table, unsigned pages, unsigned max_t, unsigned max_k, int* hits, int* fetched, int* pieces)
{
    PagedPlan p = {};
    p.c.table = table, p.c.pages = pages, p.c.shift = 4, p.c.slots = slots, p.c.ld_table = cap / 16, p.c.Hkv = Hkv, p.c.cap = cap;
    p.b.slot = slot, p.b.pos = pos, p.b.start = start, p.b.n = n, p.b.floor = floor, p.b.e0 = e0, p.b.entries = entries, p.b.t0 = t0, p.b.tokens = tokens, p.b.max_n = max_n;
    p.G = G, p.window = window, p.first = first, p.least = least;
    switch (shape)
    {
%s
    }
    return -1;
}
extern "C" int page_of(const int* table, unsigned pages, unsigned slots, unsigned ld, int slot, unsigned at)
{
    PagedCache c = {};
    c.table = table, c.pages = pages, c.slots = slots, c.ld_table = ld, c.shift = 4;
    return paged_page(c, slot, at);
}
''' % (ROOT, "\n".join("    case %d: return walk<%d, %d>(p, grid, max_t, max_k, hits, fetched, pieces);" % (i, u, r) for i, (u, r) in enumerate(SHAPES))))
    so = str(top / "plan.so")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-o", so, str(top / "plan.cpp")])
    return C.CDLL(so)


def ints(v):
    a = np.ascontiguousarray(v, np.int32)
    return a, a.ctypes.data_as(C.c_void_p)


BATCHES = {
    "one token": ([(0, 0, 1)], None),
    "decoding": ([(3, 499, 1), (0, 0, 1), (1, 16, 1), (2, 33, 1)], None),
    "ragged": ([(0, 31, 3), (2, 0, 0), (1, 200, 40), (3, 511, 1), (2, 5, 17)], None),
    "floors": ([(0, 100, 5), (1, 300, 9), (2, 64, 1), (3, 20, 30)], [99, 200, 65, 25]),    # a row that sees nothing, and rows before a floor
    "slots that are none": ([(-1, 40, 2), (1, 40, 2), (9, 3, 4)], None),
    "past the table": ([(0, 600, 30), (1, 639, 2), (2, 700, 3)], None),
    "odd": ([(0, -5, 3), (1, 10, -2), (2, 10, 4)], None),
    "nothing": ([(0, 4, 0)], None),
}


@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (16, 4), (50, 1), (33, 40), (200, 19)])
@pytest.mark.parametrize("name", BATCHES)
def test_every_key_that_a_row_sees_is_met_once(plan, name, window, first):
    entries, floor = BATCHES[name]
    cap, slots, max_k, max_t = 640, 4, 640, 64
    n = [max(0, x) for _, _, x in entries]
    meta = [ints(v) for v in ([s for s, _, _ in entries], [p for _, p, _ in entries], np.cumsum([0] + n)[:-1], [x for _, _, x in entries])]
    fl = (None, None) if floor is None else ints(floor)
    table, tp = ints(np.arange(slots * cap // 16))
    for Hkv, G in ((1, 1), (2, 3), (1, 17)):
        want = np.zeros((len(entries), Hkv, max_t, max_k), np.int32)
        for e, (s, p, k) in enumerate(entries):
            if p < 0 or not 0 <= s < slots:
                continue
            t, j = p + np.arange(max(0, k))[:, None], np.arange(max_k)
            f = 0 if floor is None else floor[e]
            seen = (j <= t) & (j >= f)
            if window:
                seen &= (j > t - window) | (j < f + first)
            want[e, :, :max(0, k)] = seen
        for shape in range(len(SHAPES)):
            for grid, least in ((1, 1), (7, 1), (148, 1), (148, 5), (1000, 8)):
                hits, fetched, pieces = np.zeros_like(want), np.zeros((len(entries), Hkv, max_k), np.int32), np.zeros(1, np.int32)
                bad = plan.run(shape, *(m[1] for m in meta), fl[1], len(entries), 0, max(1, sum(n)), 0, 64, slots, cap, Hkv, G, window, first, least, grid, tp,
                               len(table), max_t, max_k, *(a.ctypes.data_as(C.c_void_p) for a in (hits, fetched, pieces)))
                assert bad == 0, (shape, grid, least, Hkv, G)
                assert np.array_equal(hits, want), (shape, grid, least, Hkv, G)
                assert not np.any(fetched[~want.any(2)]), "a row that nobody sees is fetched"


def test_tokens_of_other_calls_are_left_alone(plan):
    """Entries whose rows lie outside the call's tokens, or go on behind them, and more tokens than max_n."""
    meta = [ints(v) for v in ([0, 1, 2], [10, 10, 10], [0, 5, 12], [5, 9, 4])]
    table, tp = ints(np.arange(160))
    hits, fetched, pieces = np.zeros((3, 1, 16, 640), np.int32), np.zeros((3, 1, 640), np.int32), np.zeros(1, np.int32)
    assert plan.run(0, *(m[1] for m in meta), None, 3, 0, 7, 5, 6, 4, 640, 1, 1, 0, 0, 1, 9, tp, 160, 16, 640,
                    *(a.ctypes.data_as(C.c_void_p) for a in (hits, fetched, pieces))) == 0
    tokens = hits.any(3)[:, 0].sum(1)
    assert tokens.tolist() == [0, 6, 0]


def test_pages_that_are_none(plan):
    t, tp = ints([[3, -1, 7, 2], [0, 8, 1 << 30, -(1 << 31)]])
    page = lambda slot, at: plan.page_of(tp, 8, 2, 4, slot, at)    # noqa: E731
    assert [page(0, 16 * i + 15) for i in range(4)] == [3, -1, 7, 2] and [page(1, 16 * i) for i in range(4)] == [0, -1, -1, -1]
    assert page(0, 64) == -1 and page(0, 0xFFFFFFFF) == -1 and page(-1, 0) == -1


# ---- refusals ------------------------------------------------------------------------------------------------------
def _calls():
    D = load_package().decoder_capi
    at = 0x10000    # never followed: the calls are refused before anything is launched
    c = dict(k=at, v=at, k_scale=at, v_scale=at, table=at, pages=9, page=16, slots=3, ld_table=4, Hkv=2, dim=64, vdim=64, k_ld=64, v_ld=64, type=4)
    a = dict(q=at, out=at, work=at, work_bytes=1 << 40, ldq=256, ldo=256, H=4, scale=1.0)
    b = dict(slot=at, pos=at, start=at, n=at, token_entry=at, entries=1, tokens=1, max_n=1, max_len=1)
    return D, c, a, b


BAD_PAGES = [dict(k=None), dict(v=None), dict(table=None), dict(k=0x10008), dict(v=0x10001), dict(page=8), dict(page=24), dict(page=0), dict(Hkv=0), dict(dim=0),
             dict(vdim=0), dict(dim=257, k_ld=272), dict(vdim=257, v_ld=272), dict(k_ld=48), dict(v_ld=72), dict(k_ld=63), dict(type=0), dict(type=5),
             dict(k_scale=None), dict(v_scale=None), dict(k_scale=0x10004), dict(v_scale=0x10002), dict(ld_table=1 << 27), dict(pages=0), dict(pages=1 << 31), dict(page=1 << 30, ld_table=0)]


@pytest.mark.parametrize("bad", BAD_PAGES, ids=str)
def test_refused_caches(bad):
    D, c, a, b = _calls()
    pages, batch = D.fill(D.Pages, **(c | bad)), D.fill(D.Batch, **b)
    assert D.lib().cuda_b200_pages_append(3, C.byref(pages), 0x10000, 128, 0x10000, 128, C.byref(batch), None, 0) == -1
    assert D.lib().cuda_b200_pages_read(3, C.byref(pages), 0x10000, 128, 0x10000, 128, C.byref(batch), None, 0) == -1
    assert D.lib().cuda_b200_paged_attention_rows(3, C.byref(D.fill(D.PagedAttention, **a)), C.byref(pages), C.byref(batch), None, 0, 0) == -1


@pytest.mark.parametrize("bad", [dict(slot=None), dict(pos=None), dict(start=None), dict(n=None), dict(first_token=0x7FFFFFFF), dict(first_entry=0x7FFFFFFF)], ids=str)
def test_refused_batches(bad):
    D, c, a, b = _calls()
    pages, batch = D.fill(D.Pages, **c), D.fill(D.Batch, **(b | bad))
    assert D.lib().cuda_b200_pages_append(3, C.byref(pages), 0x10000, 128, 0x10000, 128, C.byref(batch), None, 0) == -1
    assert D.lib().cuda_b200_paged_attention_rows(3, C.byref(D.fill(D.PagedAttention, **a)), C.byref(pages), C.byref(batch), None, 0, 0) == -1


def test_refused_arguments():
    D, c, a, b = _calls()
    L, pages, batch = D.lib(), D.fill(D.Pages, **c), D.fill(D.Batch, **b)
    for k, ldk, v, ldv, dtype in ((None, 128, 0x10000, 128, 3), (0x10000, 127, 0x10000, 128, 3), (0x10000, 128, None, 128, 3), (0x10000, 128, 0x10000, 100, 3),
                                  (0x10000, 128, 0x10000, 128, 2)):
        assert L.cuda_b200_pages_append(dtype, C.byref(pages), k, ldk, v, ldv, C.byref(batch), None, 0) == -1
        assert L.cuda_b200_pages_read(dtype, C.byref(pages), k, ldk, v, ldv, C.byref(batch), None, 0) == -1
    no_entry = D.fill(D.Batch, **(b | dict(token_entry=None)))
    assert L.cuda_b200_pages_append(3, C.byref(pages), 0x10000, 128, 0x10000, 128, C.byref(no_entry), None, 0) == -1
    many = D.fill(D.Batch, **(b | dict(tokens=1 << 30)))
    assert L.cuda_b200_pages_append(3, C.byref(pages), 0x10000, 128, 0x10000, 128, C.byref(many), None, 0) == -1
    for bad in (dict(q=None), dict(out=None), dict(work=None), dict(work=0x10008), dict(H=0), dict(H=3), dict(ldq=255), dict(ldo=255)):
        assert L.cuda_b200_paged_attention_rows(3, C.byref(D.fill(D.PagedAttention, **(a | bad))), C.byref(pages), C.byref(batch), None, 0, 0) == -1, bad
    at = C.byref(D.fill(D.PagedAttention, **a))
    assert L.cuda_b200_paged_attention_rows(2, at, C.byref(pages), C.byref(batch), None, 0, 0) == -1
    assert L.cuda_b200_paged_attention_rows(3, at, C.byref(pages), C.byref(batch), None, 0, 9) == -1
    assert L.cuda_b200_paged_attention_rows(3, at, C.byref(pages), C.byref(batch), None, 0, -1) == -1
    assert L.cuda_b200_paged_attention_rows(3, at, C.byref(pages), C.byref(D.fill(D.Batch, **(b | dict(max_n=1 << 31)))), None, 0, 0) == -1
    assert L.cuda_b200_paged_attention_rows(3, None, C.byref(pages), C.byref(batch), None, 0, 0) == -1
    assert L.cuda_b200_paged_attention_rows(3, at, None, C.byref(batch), None, 0, 0) == -1
    # nothing to do is no error
    for empty in (dict(tokens=0), dict(entries=0)):
        none = D.fill(D.Batch, **(b | empty))
        assert L.cuda_b200_pages_append(3, C.byref(pages), 0x10000, 128, 0x10000, 128, C.byref(none), None, 0) == 0
        assert L.cuda_b200_paged_attention_rows(3, at, C.byref(pages), C.byref(none), None, 0, 0) == 0
    for H, Hkv, vdim in ((3, 2, 64), (0, 1, 64), (4, 0, 64), (4, 2, 0), (4, 2, 257)):
        assert D.paged_attention_work_bytes(H, Hkv, vdim, 1) == 0
