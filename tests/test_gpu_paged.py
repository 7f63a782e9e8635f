"""The paged cache on the GPU: rows written (as they are, or in E4M3 with a power of two per row), read back, and attention over
them, against plain implementations in 64 bits."""
import numpy as np
import pytest

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu
FLOAT, BF16, E4M3 = 0, 3, 4
PLAIN, FEW, MANY = 1, 2, 3


@pytest.fixture(scope="module")
def D():
    return load_package().decoder_capi


def torch_type(t):
    import torch

    return {FLOAT: torch.float32, BF16: torch.bfloat16, E4M3: torch.float8_e4m3fn}[t]


def dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def up16(n):
    return (n + 15) // 16 * 16


def e4m3(x):
    """Codes and exponent bytes of rows of floats, and the values that they stand for, in 64 bits from the definition."""
    x = np.asarray(x, np.float64)
    fine = np.isfinite(x)
    top = np.max(np.where(fine, np.abs(x), 0), -1, keepdims=True)
    m, e = np.frexp(top / 448)
    k = np.where(top == 0, 0, np.maximum(np.where(m == 0.5, e - 1, e), -126))
    y = np.clip(np.where(np.isnan(x), 0, x) * 2.0 ** -k.astype(float), -448, 448)
    step = 2.0 ** (np.frexp(np.maximum(np.abs(y), 2.0 ** -6))[1] - 4.0)
    y = np.where(np.isnan(x), np.nan, np.round(y / step) * step)
    return y, (k[..., 0] + 127).astype(np.uint8), y * 2.0 ** k


class Cache:
    """Pages in an order of their own; whatever nobody has written is no number, with an exponent byte that is none either."""

    def __init__(self, D, dtype, type_, Hkv, dim, vdim, page=16, slots=4, rows=640, seed=0, spare=3):
        import torch

        rng = np.random.default_rng(seed)
        self.D, self.dtype, self.type, self.Hkv, self.page = D, dtype, type_, Hkv, page
        per = -(-rows // page)
        self.pages, self.slots, self.ld = slots * per + spare, slots, per
        self.table = rng.permutation(self.pages)[:slots * per].reshape(slots, per).astype(np.int32)
        self.width = dict(k=dim, v=vdim)
        self.x, self.scale = {}, {}
        for name, w in self.width.items():
            shape = (self.pages, Hkv, page, up16(w))
            if type_ == E4M3:
                self.x[name] = torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda")
                self.scale[name] = torch.full(shape[:3], 255, dtype=torch.uint8, device="cuda")
            else:
                self.x[name], self.scale[name] = torch.full(shape, float("nan"), dtype=torch_type(type_), device="cuda"), None

    def fill(self, **kw):
        self.d_table = dev(self.table)
        f = dict(k=self.x["k"], v=self.x["v"], k_scale=self.scale["k"], v_scale=self.scale["v"], table=self.d_table, pages=self.pages, page=self.page, slots=self.slots,
                 ld_table=self.ld, Hkv=self.Hkv, dim=self.width["k"], vdim=self.width["v"], k_ld=up16(self.width["k"]), v_ld=up16(self.width["v"]), type=self.type)
        return self.D.fill(self.D.Pages, **(f | kw))

    def put(self, name, slot, first, rows):
        """Rows [n][Hkv][width] from position `first` on, by plain indexing; returns the values that the cache then stands for."""
        import torch

        w = self.width[name]
        pad = np.zeros(rows.shape[:2] + (up16(w),))
        pad[..., :w] = rows
        t = first + np.arange(len(rows))
        at = self.table[slot][t // self.page].astype(np.int64)
        page, row = dev(at), dev(t % self.page)
        if self.type == E4M3:
            y, b, value = e4m3(pad)
            self.x[name][page, :, row] = dev(y).to(torch.float8_e4m3fn).view(torch.uint8)
            self.scale[name][page, :, row] = dev(b)
        else:
            new = dev(pad).to(torch_type(self.type))
            self.x[name][page, :, row] = new
            value = new.double().cpu().numpy()
        return value[..., :w]

    def bytes(self):
        return {n: (self.x[n].contiguous().view(-1).view(__import__("torch").uint8).cpu().numpy().copy(), None if self.scale[n] is None else self.scale[n].cpu().numpy().copy())
                for n in ("k", "v")}


def batch(D, entries, floor=None, start=None, **kw):
    """entries: (slot, pos, n).  Returns the description and what has to live as long."""
    n = [max(0, k) for _, _, k in entries]
    start = list(np.cumsum([0] + n)[:-1]) if start is None else start
    tokens = kw.pop("tokens", max([s + k for s, k in zip(start, n)] + [0]))
    token_entry = np.full(max(1, tokens), -1, np.int32)
    for e, (s, k) in enumerate(zip(start, n)):
        token_entry[s:s + k] = e
    keep = [dev(np.array(v, np.int32)) for v in ([s for s, _, _ in entries], [p for _, p, _ in entries], start, [k for _, _, k in entries], token_entry)]
    if floor is not None:
        keep.append(dev(np.array(floor, np.int32)))
        kw["floor"] = keep[-1]
    f = dict(slot=keep[0], pos=keep[1], start=keep[2], n=keep[3], token_entry=keep[4], entries=len(entries), tokens=tokens, max_n=max(n + [1]),
             max_len=max([p + k for _, p, k in entries]))
    return D.fill(D.Batch, **(f | kw)), keep


# ---- writing and reading -------------------------------------------------------------------------------------------
ROWS = [(0, 3, 5), (2, 0, 33), (1, 639, 1), (3, 31, 2)]


def rows_in(rng, tokens, Hkv, width, dtype, ld, off=0):
    """[tokens][ld] with rows of unequal size; a row of zeros, one with infinities, one with a NaN, tiny and huge ones."""
    import torch

    x = rng.standard_normal((tokens, Hkv, width)) * np.exp2(rng.integers(-20, 20, (tokens, Hkv, 1)))
    x[0, 0] = 0
    x[1, 0, 0], x[1, 0, -1] = np.inf, -np.inf
    x[2, 0, width // 2] = np.nan
    x[3, 0] = np.inf
    x[4, 0], x[5, 0] = 1e-38 * rng.standard_normal(width), 1e38 * rng.standard_normal(width)
    x[6, 0], x[7, 0] = 1e-42, 448.0 * 2 ** 3       # smaller than any power of two that there is; exactly the largest code
    x[8, 0, 0] = 450.0 if dtype == BF16 else 448.0001    # the next power of two
    t = torch.full((tokens * ld + off,), 7.0, dtype=torch_type(dtype), device="cuda")
    v = t[off:].view(tokens, ld)
    v[:, :Hkv * width] = dev(x.reshape(tokens, -1)).to(v.dtype)
    return v, v[:, :Hkv * width].double().cpu().numpy().reshape(tokens, Hkv, width)


@pytest.mark.parametrize("dtype,type_", [(BF16, E4M3), (BF16, BF16), (FLOAT, E4M3), (FLOAT, FLOAT)])
@pytest.mark.parametrize("Hkv,dim,vdim,page,extra,off", [(8, 128, 128, 16, 0, 0), (1, 64, 256, 32, 0, 0), (3, 80, 16, 64, 8, 0), (2, 13, 100, 16, 5, 1), (5, 250, 1, 128, 0, 3),
                                                         (32, 8, 24, 16, 16, 8)])
def test_rows_are_written_and_read_back(D, dtype, type_, Hkv, dim, vdim, page, extra, off):
    import torch

    rng = np.random.default_rng(dim + page)
    c = Cache(D, dtype, type_, Hkv, dim, vdim, page)
    other = Cache(D, dtype, type_, Hkv, dim, vdim, page)
    b, keep = batch(D, ROWS)
    tokens = sum(n for _, _, n in ROWS)
    new = {n: rows_in(rng, tokens, Hkv, w, dtype, Hkv * w + extra, off) for n, w in c.width.items()}
    pages = c.fill()
    assert D.pages_append(dtype, pages, new["k"][0], Hkv * dim + extra, new["v"][0], Hkv * vdim + extra, b) == 0 and D.check() == 0
    want, at = {n: [] for n in new}, 0
    for slot, p, n in ROWS:
        for name in new:
            want[name].append(other.put(name, slot, p, new[name][1][at:at + n]))
        at += n
    got, plain = c.bytes(), other.bytes()
    for name in new:
        a, b_ = (x[name][0] for x in (got, plain))
        if type_ == E4M3:    # any NaN is one
            same = (a == b_) | ((a & 0x7F == 0x7F) & (b_ & 0x7F == 0x7F))
            assert np.all(same) and np.array_equal(got[name][1], plain[name][1])
        else:
            x, y = (t.view({BF16: np.uint16, FLOAT: np.uint32}[type_]) for t in (a, b_))
            nan = {BF16: (0x7FFF, 0x7F80), FLOAT: (0x7FFFFFFF, 0x7F800000)}[type_]
            assert np.all((x == y) | (((x & nan[0]) > nan[1]) & ((y & nan[0]) > nan[1])))
    # and back; rows of other tokens stay
    out = {n: torch.full((tokens + 2, Hkv * w + extra), 5.0, dtype=torch_type(dtype), device="cuda") for n, w in c.width.items()}
    assert D.pages_read(dtype, pages, out["k"], Hkv * dim + extra, out["v"], Hkv * vdim + extra, b) == 0 and D.check() == 0
    for name, w in c.width.items():
        x = out[name].double().cpu().numpy()
        assert np.all(x[tokens:] == 5) and np.all(x[:, Hkv * w:] == 5)
        value = np.concatenate(want[name])
        value = dev(value).to(torch_type(dtype)).double().cpu().numpy()    # exact but for the smallest and largest numbers of the type
        assert np.array_equal(x[:tokens, :Hkv * w].reshape(value.shape), value, equal_nan=True)


@pytest.mark.parametrize("dtype,type_", [(BF16, E4M3), (BF16, BF16), (FLOAT, FLOAT)])
def test_rows_without_a_place(D, dtype, type_):
    """Entries of other calls, places that are none, tokens of no entry: nothing is written; what is read is zero, or left."""
    import torch

    c = Cache(D, dtype, type_, 2, 32, 48)
    c.table[1, 2], c.table[1, 3] = -1, c.pages
    rng = np.random.default_rng(0)
    entries = [(0, 0, 4), (1, 30, 40), (7, 0, 3), (-1, 0, 3), (2, 638, 5), (3, -2, 4), (0, 10, 2)]
    b, keep = batch(D, entries, first_entry=0)
    b.entries = 6    # the last one is another call's
    tokens = sum(n for _, _, n in entries)
    k, v = (torch.from_numpy(rng.standard_normal((tokens, 2 * w))).cuda().to(torch_type(dtype)) for w in (32, 48))
    before = c.bytes()
    pages = c.fill()
    assert D.pages_append(dtype, pages, k, 64, v, 96, b) == 0 and D.check() == 0
    other = Cache(D, dtype, type_, 2, 32, 48)
    for name, x, w in (("k", k, 32), ("v", v, 48)):
        x = x.double().cpu().numpy().reshape(tokens, 2, w)
        other.put(name, 0, 0, x[:4])
        other.put(name, 1, 30, x[4:6])
        other.put(name, 1, 64, x[4 + 34:4 + 40])
        other.put(name, 2, 638, x[50:52])
    for name in ("k", "v"):
        assert np.array_equal(c.bytes()[name][0], other.bytes()[name][0]) and not np.array_equal(c.bytes()[name][0], before[name][0])
    ko, vo = torch.full_like(k, 9), torch.full_like(v, 9)
    assert D.pages_read(dtype, pages, ko, 64, vo, 96, b) == 0 and D.check() == 0
    live = np.zeros(tokens, bool)
    live[:6] = live[38:44] = live[50:52] = True
    for o, x in ((ko, k), (vo, v)):
        o, x = o.double().cpu().numpy(), x.double().cpu().numpy()
        assert np.all(o[-2:] == 9) and np.all(o[:-2][~live[:-2]] == 0)
        if type_ != E4M3:
            assert np.array_equal(o[live], x[live])


# ---- attention -----------------------------------------------------------------------------------------------------
class Attention:
    """Queries over a cache that holds `pos + n` rows of every sequence, and the same in 64 bits."""

    def __init__(self, D, dtype, type_, H, Hkv, dim, vdim, entries, page=16, window=0, first=0, sink=False, floor=None, seed=0, scale=None, rows=640, slots=4, loud=1.0):
        import torch

        rng = np.random.default_rng(seed)
        self.D, self.dtype, self.H, self.G, self.dim, self.vdim, self.entries = D, dtype, H, H // Hkv, dim, vdim, entries
        self.window, self.first, self.floor, self.scale = window, first, floor, scale or dim ** -0.5
        self.c = Cache(D, dtype, type_, Hkv, dim, vdim, page, slots, rows, seed)
        self.T = sum(max(0, n) for _, _, n in entries)
        self.values = {}
        for e, (s, p, n) in enumerate(entries):
            f = 0 if floor is None else floor[e]
            if not 0 <= s < slots or p < 0:
                continue
            end = min(p + max(n, 0), self.c.ld * page)
            old = self.values.get(s, (np.zeros((0, Hkv, dim)), np.zeros((0, Hkv, vdim))))
            k, v = (np.zeros((max(end, len(old[0])), Hkv, w)) for w in (dim, vdim))
            k[:len(old[0])], v[:len(old[1])] = old[0], old[1]
            # rows below the floor are nobody's, and with a window those that none of the entry's tokens sees
            t = p + np.arange(max(n, 0))[:, None]
            seen = self.seen(t, np.arange(end), f).any(0)
            for j in np.flatnonzero(seen & ~np.isin(np.arange(end), self.values.get(s, ((), (), ()))[2])):
                x, y = rng.standard_normal((1, Hkv, dim)), loud ** rng.uniform(-1, 1) * rng.standard_normal((1, Hkv, vdim))
                k[j], v[j] = self.c.put("k", s, j, x)[0], self.c.put("v", s, j, y)[0]
            mine = np.flatnonzero(seen)
            self.values[s] = (k, v, np.union1d(mine, self.values.get(s, ((), (), np.zeros(0, int)))[2]))
        q = torch.from_numpy(rng.standard_normal((max(1, self.T), H * dim))).cuda().to(torch_type(dtype))
        self.q = q
        self.sink = 2 * rng.standard_normal(H).astype(np.float32) if sink else None

    def seen(self, t, j, f):
        s = (j <= t) & (j >= f)
        if self.window:
            s &= (j > t - self.window) | (j < f + self.first)
        return s

    def run(self, kernel=0, out=None, pages=None, work=None, flags=0, desc=None, **kw):
        import torch

        D, H = self.D, self.H
        b, keep = batch(D, self.entries, floor=self.floor, **kw)
        out = torch.full((max(1, self.T) + 2, H * self.vdim + 3), -2.0, dtype=self.q.dtype, device="cuda") if out is None else out
        room = 2 * D.paged_attention_work_bytes(H, H // self.G, self.vdim, max(b.max_n, 256))
        work = torch.full((room,), 0xFF, dtype=torch.uint8, device="cuda") if work is None else work
        sink = None if self.sink is None else dev(self.sink)
        a = D.fill(D.PagedAttention, **(dict(q=self.q, out=out, work=work, sink=sink, work_bytes=work.numel(), ldq=self.q.shape[1], ldo=out.shape[1], H=H, window=self.window,
                                             first=self.first, scale=self.scale) | (desc or {})))
        pages = self.c.fill() if pages is None else pages
        assert D.paged_attention(self.dtype, a, pages, b, flags=flags, kernel=kernel) == 0 and D.check() == 0
        x = out.double().cpu().numpy()
        assert np.all(x[self.T:] == -2) and np.all(x[:, H * self.vdim:] == -2), "rows and columns that are nobody's"
        return x[:self.T, :H * self.vdim].reshape(self.T, H, self.vdim)

    def reference(self, lost=(), kernel=MANY):
        """(outputs, bound).  lost: (slot, position) of keys that are on no page.

        The bound: the output's rounding, half a step of its type; the weights' rounding (FP16, or the sum of two BF16 numbers: 2^-11 of
        each at most; on tcgen05 one BF16 number, so that sum |dw v| <= 2^-8 sum |w v|), on the sum of |weight * value|; and, on the same,
        what a score may be off: products and sums of dim terms in 32 bits, (dim + 8) * 2^-24 of the sum of |q k| * scale, twice
        (numerator and denominator), with as much again for the exponential (2^-22) and the sums of the keys' terms (keys * 2^-24)."""
        many = kernel == MANY or (kernel == 0 and self.G * max(n for _, _, n in self.entries) > 16)    # (where that is the one taken)
        weight = 0 if self.dtype == FLOAT else 2.0 ** -8 if many else 2.0 ** -10
        q = self.q.double().cpu().numpy()[:self.T].reshape(self.T, self.H, self.dim)
        out, tol, at = np.zeros((self.T, self.H, self.vdim)), np.zeros((self.T, self.H, self.vdim)), 0
        half = 2.0 ** -24 if self.dtype == FLOAT else 2.0 ** -8
        for e, (s, p, n) in enumerate(self.entries):
            n = max(n, 0)
            if s in self.values and p >= 0:
                k, v, _ = self.values[s]
                k, v = k[:p + n], v[:p + n]
                t, j = p + np.arange(n)[:, None], np.arange(len(k))
                seen = self.seen(t, j, 0 if self.floor is None else self.floor[e]) & ~np.isin(j, [x for y, x in lost if y == s])
                for h in range(self.H):
                    a, b = k[:, h // self.G], v[:, h // self.G]
                    with np.errstate(invalid="ignore"):
                        z = np.where(seen, self.scale * q[at:at + n, h] @ a.T, -np.inf)
                    size = abs(self.scale) * (np.abs(q[at:at + n, h]) @ np.abs(a).T)
                    size = np.where(seen, size, 0).max(1, initial=0)[:, None]
                    top = z.max(1, initial=-np.inf, keepdims=True)
                    top = np.where(np.isfinite(top), top, 0)
                    w = np.exp(z - top)
                    l = w.sum(1, keepdims=True) + (np.exp(self.sink[h] - top) if self.sink is not None else 0)
                    w = np.where(seen.any(1, keepdims=True), w / np.where(l == 0, 1, l), 0)
                    out[at:at + n, h] = w @ b
                    weighted = w @ np.abs(b)
                    fine = 2.0 ** -24 * (2 * (self.dim + 8) * (1 + size) + len(k) + 16)
                    tol[at:at + n, h] = half * np.abs(out[at:at + n, h]) + weighted * (weight + 2 * fine)
            at += n
        return out, tol + 1e-30

    def check(self, kernel=0, what="", **kw):
        got = self.run(kernel, **kw)
        want, tol = self.reference(kernel=kernel)
        off = np.abs(got - want) / tol
        assert np.all(np.isfinite(got)) and off.max(initial=0) <= 1, (what, kernel, off.max(), np.unravel_index(off.argmax(), off.shape))
        return got


TYPES = [(BF16, BF16), (BF16, E4M3), (FLOAT, FLOAT), (FLOAT, E4M3)]
HEADS = [(32, 8, 128, 128, 16), (4, 4, 64, 64, 32), (7, 1, 80, 48, 64), (16, 2, 128, 64, 16), (6, 2, 13, 100, 16), (5, 1, 256, 256, 128), (24, 1, 96, 128, 32), (2, 1, 250, 1, 16)]
BATCHES = [
    [(0, 0, 1)],                                                 # a single token, a single key
    [(2, 15, 1), (0, 16, 1), (3, 499, 1), (1, 63, 1)],           # decoding: a page's last and first row
    [(1, 300, 3), (0, 0, 2), (3, 127, 5), (2, 31, 1)],           # several tokens each
    [(0, 0, 70), (2, 97, 45)],                                   # portions of prompts
]


def kinds(dtype, H, Hkv, entries):
    return [PLAIN] if dtype == FLOAT else [0, PLAIN, FEW, MANY]


@pytest.mark.parametrize("dtype,type_", TYPES)
@pytest.mark.parametrize("H,Hkv,dim,vdim,page", HEADS)
@pytest.mark.parametrize("b", range(len(BATCHES)))
def test_attention(D, dtype, type_, H, Hkv, dim, vdim, page, b):
    a = Attention(D, dtype, type_, H, Hkv, dim, vdim, BATCHES[b], page, sink=b == 1, seed=dim + b)
    for kernel in kinds(dtype, H, Hkv, BATCHES[b]):
        a.check(kernel)


@pytest.mark.parametrize("dtype,type_", TYPES[:3])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (16, 4), (64, 1), (100, 17), (150, 300), (640, 4)])
@pytest.mark.parametrize("dim", [64, 128])
def test_windows_and_first_keys(D, dtype, type_, window, first, dim):
    """Keys outside the window hold no numbers: nobody has written them."""
    entries = [(0, 0, 1), (1, 199, 1), (2, 331, 1), (3, 16, 1)]
    a = Attention(D, dtype, type_, 8, 2, dim, dim, entries, window=window, first=first, sink=True, seed=window)
    for kernel in kinds(dtype, 8, 2, entries):
        a.check(kernel)
    entries = [(0, 0, 90), (1, 180, 33), (2, 500, 3)]
    a = Attention(D, dtype, type_, 8, 2, dim, dim, entries, page=32, window=window, first=first, seed=window + 1)
    for kernel in kinds(dtype, 8, 2, entries):
        a.check(kernel)


@pytest.mark.parametrize("dtype,type_", TYPES[:3])
def test_floors_and_rows_that_see_nothing(D, dtype, type_):
    entries, floor = [(0, 100, 5), (1, 300, 9), (2, 64, 1), (3, 20, 30)], [103, 200, 65, 25]
    for window, first in ((0, 0), (40, 7)):
        a = Attention(D, dtype, type_, 8, 2, 64, 64, entries, window=window, first=first, floor=floor, sink=True, seed=window)
        for kernel in kinds(dtype, 8, 2, entries):
            got = a.check(kernel)
            assert np.all(got[:3] == 0) and np.all(got[14] == 0) and np.all(got[15:20] == 0) and np.all(np.abs(got[3:5]).max(2) > 0)


@pytest.mark.parametrize("dtype,type_", TYPES[:3])
def test_pages_and_slots_that_are_none(D, dtype, type_):
    entries = [(0, 200, 1), (1, 90, 3), (-1, 40, 2), (9, 10, 1), (2, 700, 1), (3, 639, 1)]
    a = Attention(D, dtype, type_, 8, 2, 64, 64, entries, seed=3)
    t = a.c.table
    t[0, 3], t[0, 12], t[1, 0], t[1, 5], t[3, :39] = -1, a.c.pages, 1 << 30, -7, -1
    lost = [(0, j) for j in (*range(48, 64), *range(192, 208))] + [(1, j) for j in (*range(16), *range(80, 96))] + [(3, j) for j in range(624)]
    want, tol = a.reference(lost)
    for kernel in kinds(dtype, 8, 2, entries):
        got = a.run(kernel)
        assert np.all(got[4:7] == 0)
        assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("type_", [BF16, E4M3])
@pytest.mark.parametrize("n", [1, 40])
def test_unequal_rows_of_values(D, type_, n):
    """Values whose sizes differ by 2^24 and keys that decide between them."""
    a = Attention(D, BF16, type_, 4, 1, 64, 64, [(0, 300 - n, n), (1, 17, n)], loud=4096.0, scale=0.7, seed=n)
    for kernel in kinds(BF16, 4, 1, a.entries):
        a.check(kernel)


@pytest.mark.parametrize("dtype,type_", TYPES[:3])
def test_one_key_far_above_the_others(D, dtype, type_):
    """Scores that grow by far more than a running maximum may without rescaling, at every place in a sequence."""
    for spot in (0, 1, 15, 16, 31, 32, 63, 64, 127, 128, 255, 300, 338):
        for n in (1, 40):
            a = Attention(D, dtype, type_, 4, 1, 64, 64, [(0, 339 - n + 1, n)], scale=1.0, seed=spot)
            k, v, _ = a.values[0]
            u = np.zeros((1, 1, 64))
            u[..., 5] = 32.0
            k[spot], v[spot] = a.c.put("k", 0, spot, u)[0], a.c.put("v", 0, spot, 3 + 0 * u)[0]
            a.q[:, 5::64] = 4.0
            for kernel in kinds(dtype, 4, 1, a.entries):
                a.check(kernel, spot)


@pytest.mark.parametrize("dtype,type_", TYPES[:3])
def test_values_that_are_no_numbers_reach_their_rows(D, dtype, type_):
    """A NaN among the values of a key that a token sees shows in its output, a score that is none makes its row none; other heads and sequences stay."""
    a = Attention(D, dtype, type_, 8, 2, 64, 64, [(0, 120, 1), (1, 80, 1)], seed=1)
    want, tol = a.reference()
    bad = a.values[0][1][30:31].copy()
    bad[0, 1, 7] = np.nan
    a.c.put("v", 0, 30, bad)
    bad = a.values[1][0][9:10].copy()
    bad[0, 0, 3] = np.nan
    a.c.put("k", 1, 9, bad)
    for kernel in kinds(dtype, 8, 2, a.entries):
        got = a.run(kernel)
        none = np.isnan(got)
        assert np.all(none[0, 4:, 7]) and none[0].sum() == 4 and np.all(none[1, :4]) and none[1].sum() == 4 * 64
        assert np.all(np.abs(got - want)[~none] <= tol[~none])


def test_scores_of_minus_infinity(D):
    """A row whose scores are all minus infinity gives zeros; beside others such a key weighs nothing."""
    a = Attention(D, BF16, BF16, 4, 1, 64, 64, [(0, 70, 1), (1, 70, 1)], sink=True, seed=2)
    low = np.full((1, 1, 64), -np.inf)
    low[..., 1:] = 0
    a.q[:] = abs(a.q) + 1
    k0, v0, _ = a.values[0]
    k1, _, _ = a.values[1]
    want_all, tol_all = None, None
    for j in range(71):
        k0[j] = a.c.put("k", 0, j, low)[0]
    for j in range(0, 71, 2):
        k1[j] = a.c.put("k", 1, j, low)[0]
    finite = k1.copy()
    a.values[1] = (np.where(np.isfinite(finite), finite, -1e4), a.values[1][1], a.values[1][2])    # exp of that is 0 too
    a.values[0] = (np.zeros_like(k0), v0, a.values[0][2])
    want_all, tol_all = a.reference()
    k = a.values[1][0]
    for kernel in kinds(BF16, 4, 1, a.entries):
        got = a.run(kernel)
        assert np.all(got[0] == 0)
        assert np.all(np.abs(got[1] - want_all[1]) <= 2.0 ** -7 * np.abs(want_all[1]) + 2.0 ** -9) and np.all(np.isfinite(got)) and k.shape[0] == 71


@pytest.mark.parametrize("dtype,type_", TYPES[:3])
@pytest.mark.parametrize("scale", [-0.3, 1e-30])
def test_scales_below_and_next_to_zero(D, dtype, type_, scale):
    a = Attention(D, dtype, type_, 8, 2, 64, 64, [(0, 130, 1), (1, 60, 25)], scale=scale, sink=True, seed=14)
    a.sink[3] = -np.inf    # a sink that takes nothing
    for kernel in kinds(dtype, 8, 2, a.entries):
        a.check(kernel, scale)


@pytest.mark.parametrize("dtype,type_", TYPES[:3])
def test_a_query_that_is_no_number_spoils_its_own_rows(D, dtype, type_):
    a = Attention(D, dtype, type_, 8, 2, 64, 64, [(0, 130, 1), (1, 60, 25)], seed=15)
    want, _ = a.reference()
    a.q[4, 2 * 64 + 5] = float("nan")
    for kernel in kinds(dtype, 8, 2, a.entries):
        got = a.run(kernel)
        none = np.isnan(got)
        assert np.all(none[4, 2]) and none.sum() == 64
        tol = np.nan_to_num(a.reference(kernel=kernel)[1], nan=1.0)
        assert np.all(np.abs(got - want)[~none] <= tol[~none]), kernel


@pytest.mark.parametrize("type_", [BF16, E4M3])
def test_one_long_sequence(D, type_):
    """Shares of every CTA in one segment."""
    a = Attention(D, BF16, type_, 4, 1, 64, 64, [(0, 6000, 1), (1, 5, 1)], rows=6016, slots=2, seed=4)
    for kernel in kinds(BF16, 4, 1, a.entries):
        got = a.check(kernel)
        assert np.array_equal(got, a.run(kernel)), "the same call gives the same bits"
    a = Attention(D, BF16, type_, 8, 1, 128, 128, [(0, 2500, 37)], rows=2560, slots=2, page=64, seed=5)
    for kernel in kinds(BF16, 8, 1, a.entries):
        got = a.check(kernel)
        assert np.array_equal(got, a.run(kernel))


def test_many_short_sequences(D):
    """More entries than a CTA has threads, most of them without tokens."""
    entries = [(i % 4, 20 * (i % 4) + 3, 1 if i % 7 else 0) for i in range(700)]
    a = Attention(D, BF16, E4M3, 4, 2, 64, 64, entries, seed=6)
    for kernel in kinds(BF16, 4, 2, entries):
        a.check(kernel)


def test_a_part_of_a_batch(D):
    """first_entry and first_token: other entries' rows stay."""
    entries = [(0, 30, 2), (1, 100, 3), (2, 64, 1), (3, 9, 4)]
    a = Attention(D, BF16, E4M3, 4, 2, 64, 64, entries, seed=7)
    want, tol = a.reference()
    for kernel in kinds(BF16, 4, 2, entries):
        got = a.run(kernel, first_entry=1, first_token=2, tokens=4)
        assert np.all(got[:2] == -2) and np.all(got[6:] == -2)
        assert np.all(np.abs(got - want)[2:6] <= tol[2:6])


def test_strides_and_odd_places(D):
    """Queries and outputs at places that cannot be accessed in vectors."""
    import torch

    for type_ in (BF16, E4M3):
        a = Attention(D, BF16, type_, 4, 2, 64, 64, [(0, 100, 1), (1, 7, 2), (2, 40, 60)], seed=8)
        wide = torch.full((a.T * 259 + 8,), 7.0, dtype=torch.bfloat16, device="cuda")[1:1 + a.T * 259].view(a.T, 259)
        wide[:, :256] = a.q[:a.T]
        a.q_plain, a.q = a.q, wide
        for kernel in kinds(BF16, 4, 2, a.entries):
            out = torch.full(((a.T + 2) * 261 + 1,), -2.0, dtype=torch.bfloat16, device="cuda")[1:].view(a.T + 2, 261)
            got = a.run(kernel, out=out)
            a.q = a.q_plain
            want, tol = a.reference()
            a.q = wide
            assert np.all(np.abs(got - want) <= tol), (type_, kernel)


def test_offsets_past_32_bits(D):
    """A cache of more than 2^32 bytes whose last pages are in use."""
    import torch

    pages, page, dim = (1 << 32) // (16 * 256) + 40, 16, 256
    for type_ in (E4M3, BF16):
        k, v = (torch.empty((pages, 1, page, dim), dtype=torch.uint8 if type_ == E4M3 else torch.bfloat16, device="cuda") for _ in range(2))
        small = Attention(D, BF16, type_, 4, 1, dim, dim, [(0, 100, 1), (1, 30, 60)], slots=2, rows=128, seed=9)
        want, tol = small.reference()
        n = small.c.pages
        k[-n:], v[-n:] = small.c.x["k"], small.c.x["v"]
        big = {}
        if type_ == E4M3:
            ks, vs = (torch.zeros((pages, 1, page), dtype=torch.uint8, device="cuda") for _ in range(2))
            ks[-n:], vs[-n:] = small.c.scale["k"], small.c.scale["v"]
            big = dict(k_scale=ks, v_scale=vs)
        small.c.table += pages - n
        desc = small.c.fill(k=k, v=v, pages=pages, **big)
        for kernel in kinds(BF16, 4, 1, small.entries):
            got = small.run(kernel, pages=desc)
            assert np.all(np.abs(got - want) <= tol)
        b, keep = batch(D, [(1, 120, 8)])
        new = torch.randn(8, dim, device="cuda").bfloat16()
        got = [torch.zeros_like(new) for _ in range(2)]
        assert D.pages_append(BF16, desc, new, dim, new, dim, b) == 0 and D.pages_read(BF16, desc, got[0], dim, got[1], dim, b) == 0 and D.check() == 0
        value = e4m3(new.double().cpu().numpy())[2] if type_ == E4M3 else new.double().cpu().numpy()
        assert all(np.array_equal(x.double().cpu().numpy(), value) for x in got)
        del k, v


def test_too_little_scratch_is_refused(D):
    import torch

    a = Attention(D, BF16, E4M3, 4, 2, 64, 64, [(0, 30, 2)], seed=1)
    b, keep = batch(D, a.entries)
    out = torch.zeros(a.T, 256, dtype=torch.bfloat16, device="cuda")
    room = D.paged_attention_work_bytes(4, 2, 64, 2)
    work = torch.zeros(room, dtype=torch.uint8, device="cuda")
    f = dict(q=a.q, out=out, work=work, ldq=256, ldo=256, H=4, scale=1.0)
    pages = a.c.fill()
    assert D.paged_attention(BF16, D.fill(D.PagedAttention, work_bytes=room - 1, **f), pages, b) == -1
    assert torch.count_nonzero(out) == 0
    assert D.paged_attention(BF16, D.fill(D.PagedAttention, work_bytes=room, **f), pages, b) == 0 and D.check() == 0
    assert torch.count_nonzero(out) > 0


# ---- together, as a server runs them -------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,type_", TYPES[:3])
def test_sequences_that_grow(D, dtype, type_):
    """Two sequences: a prompt in portions, then tokens one by one, one of them joining late; pages are handed out as they grow, and a
    shared first page is only read.  Every step's rows against the definition over all rows so far."""
    import torch

    H, Hkv, dim, vdim, page, window, first = 8, 2, 64, 48, 16, 60, 5
    rng = np.random.default_rng(11)
    c = Cache(D, dtype, type_, Hkv, dim, vdim, page, slots=3, rows=256)
    free, c.table = list(rng.permutation(c.pages)), np.full_like(c.table, -1)
    a = Attention.__new__(Attention)
    a.D, a.dtype, a.H, a.G, a.dim, a.vdim, a.window, a.first, a.floor, a.scale, a.c = D, dtype, H, H // Hkv, dim, vdim, window, first, None, dim ** -0.5, c
    a.sink = rng.standard_normal(H).astype(np.float32)
    a.values = {s: (np.zeros((0, Hkv, dim)), np.zeros((0, Hkv, vdim)), None) for s in range(3)}
    work = torch.zeros(D.paged_attention_work_bytes(H, Hkv, vdim, 64), dtype=torch.uint8, device="cuda")
    length = [0, 0, 0]
    steps = [[(0, 37)], [(0, 30), (1, 50)], [(0, 1), (1, 14)]] + [[(0, 1), (1, 1)]] * 5 + [[(1, 1), (0, 1), (2, 24)]] + [[(2, 1), (1, 1), (0, 1)]] * 3 + [[(0, 40), (2, 1)]]
    for step, news in enumerate(steps):
        if step == 8:    # the third sequence begins with the first one's first page
            c.table[2, 0] = c.table[0, 0]
            length[2] = page
            a.values[2] = tuple(x[:page].copy() for x in a.values[0][:2]) + (None,)
        a.entries = [(s, length[s], n) for s, n in news]
        for s, n in news:
            for i in range(-(-(length[s] + n) // page)):
                if c.table[s, i] < 0:
                    c.table[s, i] = free.pop()
        T = a.T = sum(n for _, n in news)
        ld = (H * dim + Hkv * (dim + vdim) + 63) // 64 * 64
        x = torch.from_numpy(rng.standard_normal((T, ld))).cuda().to(torch_type(dtype))    # q, k and v side by side, as a linear leaves them
        b, keep = batch(D, a.entries)
        pages = c.fill()
        at = lambda n: x.data_ptr() + n * x.element_size()    # noqa: E731
        assert D.pages_append(dtype, pages, at(H * dim), ld, at(H * dim + Hkv * dim), ld, b, flags=1) == 0
        a.q = x[:, :H * dim]
        out = torch.full((T, H * vdim), -2.0, dtype=x.dtype, device="cuda")
        sink = dev(a.sink)
        desc = D.fill(D.PagedAttention, q=x, out=out, work=work, sink=sink, work_bytes=work.numel(), ldq=ld, ldo=H * vdim, H=H, window=window, first=first, scale=a.scale)
        assert D.paged_attention(dtype, desc, pages, b, flags=1) == 0 and D.check() == 0
        f, row = x.double().cpu().numpy(), 0
        for s, n in news:
            k = f[row:row + n, H * dim:H * dim + Hkv * dim].reshape(n, Hkv, dim)
            v = f[row:row + n, H * dim + Hkv * dim:H * dim + Hkv * (dim + vdim)].reshape(n, Hkv, vdim)
            if type_ == E4M3:
                k, v = e4m3(k)[2], e4m3(v)[2]
            a.values[s] = (np.concatenate([a.values[s][0], k]), np.concatenate([a.values[s][1], v]), None)
            length[s] += n
            row += n
        want, tol = a.reference()
        got = out.double().cpu().numpy().reshape(T, H, vdim)
        assert np.all(np.abs(got - want) <= tol), step


def test_a_graph_whose_sequences_grow(D):
    """A captured step - write, attend - replayed with other positions and pages in its arrays, on a stream of its own, between calls of the
    same kind on another stream with scratch of their own."""
    import torch

    H, Hkv, dim, page = 8, 2, 64, 16
    c = Cache(D, BF16, E4M3, Hkv, dim, dim, page, slots=2, rows=256)
    a = Attention(D, BF16, E4M3, H, Hkv, dim, dim, [(0, 0, 1), (1, 0, 1)], seed=12)
    other = Attention(D, BF16, BF16, 4, 1, 128, 128, [(0, 500, 1), (1, 100, 30)], seed=13)
    other_want, other_tol = other.reference()
    a.c = c
    a.values = {s: (np.zeros((0, Hkv, dim)), np.zeros((0, Hkv, dim)), None) for s in range(2)}
    b, keep = batch(D, a.entries, max_len=256)
    pages = c.fill()
    x = torch.zeros(2, (H + 2 * Hkv) * dim, dtype=torch.bfloat16, device="cuda")
    ld = x.shape[1]
    out = torch.zeros(2, H * dim, dtype=torch.bfloat16, device="cuda")
    work = torch.zeros(D.paged_attention_work_bytes(H, Hkv, dim, 1), dtype=torch.uint8, device="cuda")
    desc = D.fill(D.PagedAttention, q=x, out=out, work=work, work_bytes=work.numel(), ldq=ld, ldo=H * dim, H=H, scale=a.scale)

    def step():
        return D.pages_append(BF16, pages, x.data_ptr() + H * dim * 2, ld, x.data_ptr() + (H + Hkv) * dim * 2, ld, b, flags=1) or D.paged_attention(BF16, desc, pages, b,
                                                                                                                                                 flags=1)

    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    assert step() == 0 and D.check() == 0
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        assert step() == 0
    ob, okeep = batch(D, other.entries)
    oo = torch.zeros(other.T, 512, dtype=torch.bfloat16, device="cuda")
    ow = torch.zeros(D.paged_attention_work_bytes(4, 1, 128, 30), dtype=torch.uint8, device="cuda")
    od, opages = D.fill(D.PagedAttention, q=other.q, out=oo, work=ow, work_bytes=ow.numel(), ldq=512, ldo=512, H=4, scale=other.scale), other.c.fill()
    for i in range(40):
        x.copy_(torch.randn_like(x))
        keep[1].copy_(torch.tensor([i, 3 * i], dtype=torch.int32))
        f = x.double().cpu().numpy()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
        oo.zero_()
        assert D.paged_attention(BF16, od, opages, ob) == 0
        assert D.check() == 0
        for s, p in ((0, i), (1, 3 * i)):
            k, v = (np.zeros((p + 1, Hkv, dim)) for _ in range(2))
            old = a.values[s]
            k[:len(old[0])], v[:len(old[1])] = old[0], old[1]
            k[p], v[p] = (e4m3(f[s, j:j + Hkv * dim].reshape(Hkv, dim))[2] for j in (H * dim, (H + Hkv) * dim))
            for gap in range(len(old[0]), p):    # the second sequence leaves rows out: somebody else writes them
                k[gap], v[gap] = c.put("k", s, gap, 0.1 * np.ones((1, Hkv, dim)))[0], c.put("v", s, gap, 0.1 * np.ones((1, Hkv, dim)))[0]
            a.values[s] = (k, v, None)
        a.q, a.entries, a.T = x[:, :H * dim], [(0, i, 1), (1, 3 * i, 1)], 2
        with torch.cuda.stream(stream):
            g.replay()
        torch.cuda.synchronize()
        want, tol = a.reference()
        got = out.double().cpu().numpy().reshape(2, H, dim)
        assert np.all(np.abs(got - want) <= tol), i
        assert np.all(np.abs(oo.double().cpu().numpy().reshape(other.T, 4, 128) - other_want) <= other_tol), i


def test_prompts_one_behind_the_other(D):
    """Many calls for many query rows in a row, each allowed to start before the one in front has ended: two of them fit an SM, tensor memory for one."""
    import torch

    a = Attention(D, BF16, BF16, 8, 2, 64, 64, [(0, 0, 200), (1, 300, 90)], seed=16)
    want, tol = a.reference()
    b, keep = batch(D, a.entries)
    pages = a.c.fill()
    outs = [torch.zeros(a.T, 8 * 64, dtype=torch.bfloat16, device="cuda") for _ in range(6)]
    work = torch.zeros(D.paged_attention_work_bytes(8, 2, 64, 200), dtype=torch.uint8, device="cuda")
    descs = [D.fill(D.PagedAttention, q=a.q, out=o, work=work, work_bytes=work.numel(), ldq=512, ldo=512, H=8, scale=a.scale) for o in outs]
    for _ in range(5):
        for d in descs:
            assert D.paged_attention(BF16, d, pages, b, flags=1) == 0
    assert D.check() == 0
    for o in outs:
        assert np.all(np.abs(o.double().cpu().numpy().reshape(want.shape) - want) <= tol)
