"""What the operators of the paged cache are measured on: writing keys and values of new tokens into pages (as they are, or in
8 bits with a power of two per row), reading them back, and attention of new tokens - one per sequence when decoding, many in
a prompt - over such a cache, with windows, first tokens that stay visible and sink scores.  Sizes are the benchmark's layer (32
heads, 8 of them for keys and values, 128 elements, 4096 cached rows) and generic ones around it.

Kinds of cases: append, read, attention.  `sequences` sequences hold up to `context` tokens each and get up to `tokens` more;
with `ragged` they differ in both.  `cache` says how the pages are held, `dtype` what goes in and comes out.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"bf16": (3, torch.bfloat16, 2), "float": (0, torch.float32, 4)}


def _package():
    """The package directory carries a hyphen: imported by path."""
    name = "cccc_lite_b200"
    if name not in sys.modules:
        path = os.path.join(ROOT, "cccc-lite_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(path, "__init__.py"), submodule_search_locations=[path])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


# ---- the cases -----------------------------------------------------------------------------------------------------
def _case(kind, **kw):
    c = dict(kind=kind, dtype="bf16", cache="e4m3", sequences=1, context=0, tokens=1, ragged=False, H=32, Hkv=8, dim=128, vdim=128, page=16)
    if kind == "attention":
        c |= dict(window=0, first=0, sink=False)
    return c | kw


def listed():
    return [
        # a decode step's new rows of thirty-two users: the smallest write, latency counts
        _case("append", name="append_step", sequences=32, context=4000, ragged=True),
        # a long prompt's rows at once
        _case("append", name="append_prompt", tokens=8192, page=64),
        # three short pieces moved out of the cache in float, odd lengths: the smallest read
        _case("read", name="read_pieces", dtype="float", sequences=3, context=130, tokens=77, ragged=True, page=32),
        # a long sequence taken out of the cache
        _case("read", name="read_prompt", tokens=16384, page=16),
        # the smallest attention: one user, one token, a short conversation
        _case("attention", name="decode_1", cache="bf16", context=499),
        # the benchmark's context, thirty-two users
        _case("attention", name="decode_32", sequences=32, context=4095),
        # two tokens each (one of them guessed), unequal lengths, a cache in BF16
        _case("attention", name="decode_48_ragged", cache="bf16", sequences=48, context=4000, tokens=2, ragged=True, page=32),
        # one user with a long document
        _case("attention", name="decode_long", context=131070, page=64),
        # endless conversations: a window, four first tokens that stay visible, sink scores; heads of 64
        _case("attention", name="decode_window", sequences=64, context=16000, ragged=True, H=64, dim=64, vdim=64, window=1024, first=4, sink=True),
        # a prompt from its first token on
        _case("attention", name="prompt_4096", cache="bf16", tokens=4096, page=64),
        # a portion of a prompt behind a long cached document, in 8 bits
        _case("attention", name="portion_long", context=32000, tokens=512, page=64),
        # portions of several prompts in one step, windowed
        _case("attention", name="portions_window", cache="bf16", sequences=6, context=2500, tokens=701, ragged=True, window=512, first=4, page=32),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max((work(c) for c in listed()), key=lambda w: w["bytes"] + w["flops"] / 200)
    while True:
        kind = rng.choice(["append", "read", "attention", "attention", "attention", "attention"])
        dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 128, 192, 256])
        vdim = dim if rng.random() < 0.8 else rng.choice([64, 128])
        Hkv, G = rng.choice([(8, 4), (8, 4), (8, 8), (4, 7), (2, 5), (1, 8), (16, 1), (32, 1), (8, 2)])
        dtype = "float" if rng.random() < 0.1 else "bf16"
        c = _case(kind, dtype=dtype, cache=rng.choice(["e4m3", dtype]), H=Hkv * G, Hkv=Hkv, dim=dim, vdim=vdim, page=rng.choice([16, 16, 32, 64, 128]),
                  sequences=_log_uniform(rng, 1, 64), context=_log_uniform(rng, 1, 131072) - 1, tokens=1 if rng.random() < 0.5 else _log_uniform(rng, 2, 4096),
                  ragged=rng.random() < 0.6)
        if kind != "attention":
            c["context"] = min(c["context"], 4096)
            c["tokens"] = _log_uniform(rng, 1, 16384)
        else:
            if rng.random() < 0.35:
                c |= dict(window=_log_uniform(rng, 16, 4096), first=rng.choice([0, 1, 4, 19]))
            c["sink"] = rng.random() < 0.3
        w = work(c)
        most_of = 16 if dtype == "float" and kind == "attention" else 1    # true floats have no tensor cores
        if w["bytes"] + w["flops"] / 200 > (most["bytes"] + most["flops"] / 200) / most_of:
            continue
        # what the plain form holds at once: every head's score of a padded batch, and the padded keys and values
        pos, n = _lengths(c)
        longest = max(p + k for p, k in zip(pos, n))
        if sum(pos) + sum(n) > 300000 or (kind == "attention" and len(n) * longest * max(c["H"] * max(n), 4 * Hkv * (dim + vdim)) > 1 << 30):
            continue
        return c


def _lengths(c):
    """Cached and new tokens of each sequence."""
    S = range(c["sequences"])
    if not c["ragged"]:
        return [c["context"] for _ in S], [c["tokens"] for _ in S]
    return [c["context"] - (i * 37 % 61) * c["context"] // 83 for i in S], [max(1, c["tokens"] - (i * 29 % 31) * c["tokens"] // 47) for i in S]


def _element(c):
    return 1 if c["cache"] == "e4m3" else TYPES[c["dtype"]][2]


def _seen(c, t):
    """Keys that a token at position t sees."""
    if c["window"] == 0 or t + 1 <= c["window"]:
        return t + 1
    return c["window"] + min(c["first"], t + 1 - c["window"])


def work(c):
    pos, n = _lengths(c)
    tokens, e, x = sum(n), _element(c), TYPES[c["dtype"]][2]
    row = c["Hkv"] * (c["dim"] + c["vdim"])
    held = row * e + (2 * c["Hkv"] if c["cache"] == "e4m3" else 0)
    if c["kind"] != "attention":
        return {"bytes": tokens * (row * x + held), "flops": tokens * row if c["cache"] == "e4m3" else 0}
    keys = pairs = 0
    for p, k in zip(pos, n):
        last = p + k - 1
        keys += last + 1 if c["window"] == 0 else min(last + 1, c["window"] + k - 1 + min(c["first"], max(0, p + 1 - c["window"])))
        pairs += k * (2 * p + k + 1) // 2 if c["window"] == 0 else sum(_seen(c, t) for t in range(p, p + k))
    return {"bytes": keys * held + tokens * c["H"] * (c["dim"] + c["vdim"]) * x, "flops": 2 * (c["dim"] + c["vdim"]) * c["H"] * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _ld(width):
    return (width + 15) // 16 * 16


def _rows(g, shape, loud=()):
    """Keys or values: normal, with a few loud elements and tokens of unequal size."""
    x = torch.randn(shape, generator=g, device="cuda")
    for j in loud:
        x[..., j] *= 4
    x *= torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device="cuda"))
    return x


def _quantise(x):
    """Codes (E4M3) of rows and the exponent bytes of their powers of two: the smallest one with which the row's largest element is at most 448."""
    top = x.abs().amax(-1, keepdim=True).float()
    m, e = torch.frexp(top)
    e = torch.where(top == 0, 0, (e - 9 + (m > 0.875)).clamp(-126, 127))
    return torch.ldexp(x.float(), -e).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).squeeze(-1)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    code, dtype, _ = TYPES[c["dtype"]]
    pos, n = _lengths(c)
    S, page, Hkv, dim, vdim = c["sequences"], c["page"], c["Hkv"], c["dim"], c["vdim"]
    per = [-(-(p + k) // page) for p, k in zip(pos, n)]
    pages, ld_table = sum(per) + 3, max(per) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((S, ld_table), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, k in enumerate(per):
        table[i, :k] = order[at:at + k]
        at += k
    start = [sum(n[:i]) for i in range(S)]
    tokens = sum(n)
    meta = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (list(range(S)), pos, start, n)]
    entry = torch.repeat_interleave(torch.arange(S, device="cuda", dtype=torch.int32), meta[3].long())
    s = dict(case=c, page=page, Hkv=Hkv, table=table, slot=meta[0], pos=meta[1], start=meta[2], n=meta[3], entry=entry, longest=max(p + k for p, k in zip(pos, n)),
             most=max(n), tokens=tokens, dtype=dtype)
    for name, width in (("k", dim), ("v", vdim)):
        ld = _ld(width)
        x = _rows(g, (pages, Hkv, page, ld), (3, 17) if name == "k" else ())
        x[..., width:] = 0
        if c["cache"] == "e4m3":
            s[name], s[name + "_scale"] = _quantise(x)
        else:
            s[name], s[name + "_scale"] = x.to(dtype), None
        s["new_" + name] = None
        if c["kind"] == "append":
            s["new_" + name] = _rows(g, (tokens, Hkv, width), (3, 17) if name == "k" else ()).to(dtype).view(tokens, Hkv * width)
        elif c["kind"] == "read":
            s["out_" + name] = torch.zeros(tokens, Hkv * width, dtype=dtype, device="cuda")
        del x
    if c["kind"] == "attention":
        s["scale"] = 1.0 / math.sqrt(dim)
        s["q"] = torch.randn(tokens, c["H"] * dim, generator=g, device="cuda").to(dtype)
        s["sink"] = torch.randn(c["H"], generator=g, device="cuda") if c["sink"] else None
        s["out"] = torch.zeros(tokens, c["H"] * vdim, dtype=dtype, device="cuda")
    if own:    # the descriptors and the scratch memory that a program keeps beside its cache
        D = _package().decoder_capi
        s["D"], s["code"] = D, code
        s["pages"] = D.fill(D.Pages, k=s["k"], v=s["v"], k_scale=s["k_scale"], v_scale=s["v_scale"], table=table, pages=pages, page=page, slots=S, ld_table=ld_table,
                            Hkv=Hkv, dim=dim, vdim=vdim, k_ld=_ld(dim), v_ld=_ld(vdim), type=4 if c["cache"] == "e4m3" else code)
        s["batch"] = D.fill(D.Batch, slot=meta[0], pos=meta[1], start=meta[2], n=meta[3], token_entry=entry, entries=S, tokens=tokens, max_n=s["most"],
                            max_len=s["longest"])
        if c["kind"] == "attention":
            room = D.paged_attention_work_bytes(c["H"], Hkv, vdim, s["most"])
            s["work"] = torch.empty(room, dtype=torch.uint8, device="cuda")
            s["attention"] = D.fill(D.PagedAttention, q=s["q"], out=s["out"], work=s["work"], sink=s["sink"], work_bytes=room, ldq=c["H"] * dim, ldo=c["H"] * vdim,
                                    H=c["H"], window=c["window"], first=c["first"], scale=s["scale"])
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------
def _check(rc):
    if rc != 0:
        raise RuntimeError("the call returned %d" % rc)


def _places(s):
    """Page and row of every new token."""
    e = s["entry"].long()
    p = s["pos"].long()[e] + torch.arange(s["tokens"], device="cuda") - s["start"].long()[e]
    return s["table"][s["slot"].long()[e], p // s["page"]].long(), p % s["page"]


def _append(s):
    c = s["case"]
    if own:
        _check(s["D"].pages_append(s["code"], s["pages"], s["new_k"], c["Hkv"] * c["dim"], s["new_v"], c["Hkv"] * c["vdim"], s["batch"]))
    else:
        page, row = _places(s)
        for name, width in (("k", c["dim"]), ("v", c["vdim"])):
            x = torch.nn.functional.pad(s["new_" + name].view(-1, c["Hkv"], width), (0, _ld(width) - width))
            if c["cache"] == "e4m3":
                codes, scale = _quantise(x)
                s[name].view(torch.uint8)[page, :, row] = codes.view(torch.uint8)
                s[name + "_scale"][page, :, row] = scale
            else:
                s[name][page, :, row] = x
    return {k: s[k] for k in ("k", "v", "k_scale", "v_scale")}


def _taken(s, name, width, page, row):
    """Rows of the cache as floats: [...][Hkv][width]."""
    x = s[name]
    if x.dtype == torch.float8_e4m3fn:
        two = torch.ldexp(torch.ones((), device="cuda"), s[name + "_scale"][page, :, row].int() - 127)
        return x.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn)[..., :width].float() * two[..., None]
    return x[page, :, row][..., :width].float()


def _read(s):
    c = s["case"]
    if own:
        _check(s["D"].pages_read(s["code"], s["pages"], s["out_k"], c["Hkv"] * c["dim"], s["out_v"], c["Hkv"] * c["vdim"], s["batch"]))
        return s["out_k"], s["out_v"]
    page, row = _places(s)
    return tuple(_taken(s, name, c[w], page, row).to(s["dtype"]).flatten(1) for name, w in (("k", "dim"), ("v", "vdim")))


def _attention(s):
    c = s["case"]
    if own:
        _check(s["D"].paged_attention(s["code"], s["attention"], s["pages"], s["batch"]))
        return s["out"]
    S, L, N, Hkv, G = c["sequences"], s["longest"], s["most"], c["Hkv"], c["H"] // c["Hkv"]
    # keys and values of a padded batch, one head after the other
    j = torch.arange(L, device="cuda")
    page = s["table"][s["slot"].long()][:, j // s["page"]].long().clamp_min(0)
    row = (j % s["page"]).expand(S, L)
    K, V = (_taken(s, name, c[w], page, row).transpose(1, 2) for name, w in (("k", "dim"), ("v", "vdim")))
    i = torch.arange(N, device="cuda")
    token = (s["start"].long()[:, None] + i).clamp_max(s["tokens"] - 1)
    q = s["q"].float()[token].view(S, N, Hkv, G, c["dim"]).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * N, c["dim"])
    t = s["pos"].long()[:, None] + i
    seen = j <= t[..., None]
    if c["window"]:
        seen &= (j > t[..., None] - c["window"]) | (j < c["first"])
    V = torch.where(seen.any(1)[:, None, :, None], V, 0.0)
    z = (torch.matmul(q, K.transpose(-1, -2)) * s["scale"]).view(S, Hkv, G, N, L)
    z.masked_fill_(~seen[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    z = z.sub_(top).exp_()
    total = z.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"].view(1, Hkv, G, 1, 1) - top)
    o = torch.matmul(z.view(S, Hkv, G * N, L), V).view(S, Hkv, G, N, c["vdim"]) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(S, N, c["H"] * c["vdim"])
    return o[i < s["n"][:, None]].to(s["dtype"])


def run(state):
    return {"append": _append, "read": _read, "attention": _attention}[state["case"]["kind"]](state)


# ---- the same in 64 bits -------------------------------------------------------------------------------------------
def _values(x, scale):
    """A cache's values: sign, exponent and mantissa of each code put together."""
    if scale is None:
        return x.double()
    b = x.view(torch.uint8).int()
    e, m = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (m + 8) * torch.exp2((e - 10).double()))
    return torch.where(b >= 128, -v, v) * torch.exp2(scale.double() - 127)[..., None]


def _rounded(x):
    """To the four-bit significands of E4M3 (steps of 2^-9 below 2^-6), ties to even."""
    step = torch.exp2((torch.frexp(x.abs().clamp_min(2.0 ** -6))[1] - 4).double())
    return torch.round(x / step) * step


def exact(case, seed):
    c, s = dict(case), prepare(case, seed)
    pos, n = _lengths(c)
    page, Hkv = c["page"], c["Hkv"]
    table = s["table"].cpu().tolist()

    def rows(x, i, first, last):    # [head][row][element] of sequence i
        held = x[torch.tensor(table[i][first // page:(last - 1) // page + 1], device="cuda")]
        held = held.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])
        return held[:, first % page:first % page + last - first]

    if c["kind"] == "append":
        out = {}
        for name, width in (("k", c["dim"]), ("v", c["vdim"])):
            held = s[name].double()
            new, at = s["new_" + name].double().view(-1, Hkv, width), 0
            for i, (p, k) in enumerate(zip(pos, n)):
                x = new[at:at + k]
                if c["cache"] == "e4m3":
                    top = x.abs().amax(-1, keepdim=True)
                    part, e = torch.frexp(top / 448)
                    e = (e - (part == 0.5).int()).clamp(-126, 127)
                    x = _rounded(x / torch.where(top == 0, 1.0, torch.exp2(e.double())))
                t = torch.arange(p, p + k, device="cuda")
                place = torch.tensor(table[i], device="cuda")[t // page]
                held[place, :, t % page, :width] = x
                held[place, :, t % page, width:] = 0
                at += k
            out[name], out[name + "_scale"] = held, None
        return out
    if c["kind"] == "read":
        K, V = _values(s["k"], s["k_scale"])[..., :c["dim"]], _values(s["v"], s["v_scale"])[..., :c["vdim"]]
        return tuple(torch.cat([rows(x, i, p, p + k).transpose(0, 1).flatten(1) for i, (p, k) in enumerate(zip(pos, n))]) for x in (K, V))
    if work(c)["flops"] > 1e12:
        return None
    G, got, at = c["H"] // Hkv, [], 0
    K, V = _values(s["k"], s["k_scale"]), _values(s["v"], s["v_scale"])
    for i, (p, k) in enumerate(zip(pos, n)):
        keys, values = rows(K, i, 0, p + k)[..., :c["dim"]], rows(V, i, 0, p + k)[..., :c["vdim"]]
        t, j = torch.arange(p, p + k, device="cuda")[:, None], torch.arange(p + k, device="cuda")
        hidden = j > t
        if c["window"]:
            hidden |= (j <= t - c["window"]) & (j >= c["first"])
        heads = []
        for h in range(c["H"]):
            q = s["q"][at:at + k, h * c["dim"]:(h + 1) * c["dim"]].double()
            z = torch.where(hidden, -math.inf, q @ keys[h // G].T * s["scale"])
            if s["sink"] is not None:
                z = torch.cat([z, s["sink"][h].double().expand(k, 1)], 1)
            heads.append(torch.softmax(z, 1)[:, :p + k] @ values[h // G])
        got.append(torch.stack(heads, 1).flatten(1))
        at += k
    return torch.cat(got)
