"""Performance cases of paged KV caches: many sequences' keys and values in pages of one pool.

The operators: the rows of a call, whichever sequences they belong to, rotated by their positions, normalised per head
where the model does that, and stored in their sequences' pages (xtg_hip_paged_append); a span of each sequence's rows read
back (xtg_hip_paged_read); and attention of every sequence's new rows, from one decoded token to a prompt chunk, over its
pages (xtg_hip_paged_attention).

A pool has pages of `page_size` positions for all KV heads, in BF16, in FP8 (E4M3 codes, an FP32 scale amax / 448 for each
position and KV head) or in NVFP4 (E2M1 codes, for each 16 dims an E4M3 scale nearest to amax / 6). Position p of sequence s
is in page pages[s][p // page_size]. Sequence s has rows starts[s] .. starts[s + 1] - 1 of a call, at positions pos[s] and
on. Rotation turns the pair (x_i, x_{i + d/2}) by p * theta^(-2i/d). A row at position t sees the positions p <= t of its
own sequence, and p > t - window where there is a window, with scores q.k * scale, then cap * tanh(score / cap).

Head layouts, windows, thetas and contexts are those of the two configurations of xtier-go_amd/workloads.py and of its
tests. Keys are unit vectors as attention sees them.
"""
import importlib
import math
import os
import random
import sys

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _shape(case, seqs, heads, kv_heads, d, cache, page, deal, first=0, least=1, most=1, lo=0, hi=0):
    """A call's sequences: the first has `first` rows where that is given, the others least .. most, each at a position of
    lo .. hi; `deal` draws them."""
    return dict(case, seqs=seqs, heads=heads, kv_heads=kv_heads, d=d, cache=cache, page=page, deal=deal, first=first,
                least=least, most=most, lo=lo, hi=hi)


def _append(x, theta, norm, *shape, **more):
    return _shape({"kind": "append", "x": x, "theta": theta, "norm": norm}, *shape, **more)


def _read(*shape, **more):
    return _shape({"kind": "read"}, *shape, **more)


def _attn(window, cap, *shape, **more):
    return _shape({"kind": "attn", "window": window, "cap": cap}, *shape, **more)


def listed():
    return [
        # one decoded token of one sequence, its rows as FP32 projections leave them
        dict(_append("f32", 1e6, False, 1, 32, 8, 128, "bf16", 64, 1, lo=4095, hi=4095), name="append-1row"),
        # a decode step of 64 sequences, rows normalised per head and queries scaled as the nGPT layers want them
        dict(_append("f32", 1e4, True, 64, 16, 4, 256, "fp8", 64, 2, lo=1, hi=16000), name="append-64seqs"),
        # prompts of any length that start at once
        dict(_append("bf16", 1e6, False, 9, 32, 8, 128, "bf16", 128, 3, least=17, most=900), name="append-9prompts"),
        # the last few rows of some sequences (to hand them to another pool), heads of 64 dims
        dict(_read(3, 16, 8, 64, "fp8", 32, 4, least=1, most=40, hi=3000), name="read-3seqs"),
        # a long sequence moved out of its pages, an odd number of rows
        dict(_read(1, 32, 8, 128, "nvfp4", 256, 5, first=32749, lo=13, hi=13), name="read-32749rows"),
        # two sequences that have just begun, heads of 64 dims
        dict(_attn(0, 0.0, 2, 16, 8, 64, "bf16", 32, 6, hi=40), name="attn-2seqs-short"),
        # one token of one long sequence: nothing but the split over its length fills the chip
        dict(_attn(0, 0.0, 1, 32, 8, 128, "bf16", 64, 7, lo=32767, hi=32767), name="attn-1seq-32k"),
        # a decode step of 64 sequences of any length over 8-bit pages
        dict(_attn(0, 0.0, 64, 32, 8, 128, "fp8", 64, 8, hi=8191), name="attn-64seqs-8k"),
        # a wide decode step of a sliding layer, capped scores
        dict(_attn(1024, 50.0, 256, 16, 4, 256, "bf16", 64, 9, lo=17, hi=4000), name="attn-256seqs-window"),
        # a speculative verify step of 8 rows a sequence over 4-bit pages
        dict(_attn(0, 0.0, 16, 32, 8, 128, "nvfp4", 64, 10, least=8, most=8, lo=500, hi=9000), name="attn-16seqs-verify"),
        # a prompt's chunk in the middle of it, decoded along with other sequences' single tokens
        dict(_attn(0, 0.0, 32, 32, 8, 128, "bf16", 64, 11, first=512, lo=3000, hi=6000), name="attn-chunk-and-31seqs"),
        # prompts of any length, from their beginning
        dict(_attn(0, 0.0, 4, 16, 4, 256, "fp8", 64, 12, least=150, most=1100), name="attn-4prompts"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


LAYOUTS = ((32, 8, 128), (16, 4, 256), (16, 8, 64), (32, 8, 128), (12, 4, 128))


def draw(rng):
    heads, kv_heads, d = rng.choice(LAYOUTS)
    page, deal = rng.choice([32, 64, 64, 128, 256]), rng.randint(1, 1 << 30)
    kind = rng.choice(["append", "read", "attn", "attn", "attn"])
    if kind == "append":
        cache = rng.choice(["bf16", "fp8"])
        if rng.random() < 0.5:
            rows = {"seqs": _log(rng, 1, 256), "hi": rng.choice([500, 8000])}
        else:
            rows = {"seqs": rng.randint(1, 9), "least": 1, "most": _log(rng, 2, 900), "hi": rng.choice([0, 3000])}
        return _append(rng.choice(["f32", "bf16"]), rng.choice([0.0, 1e4, 1e6, 1e7]), rng.random() < 0.5, rows.pop("seqs"), heads, kv_heads,
                       d, cache, page, deal, **rows)
    cache = rng.choice(["bf16", "fp8", "nvfp4"])
    if kind == "read":
        if rng.random() < 0.5:
            return _read(1, heads, kv_heads, d, cache, page, deal, first=_log(rng, 1, 16384), hi=3000)
        return _read(rng.randint(2, 32), heads, kv_heads, d, cache, page, deal, least=1, most=_log(rng, 2, 500), hi=3000)
    window = rng.choice([0, 0, 256, 1024])
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    shape = rng.choice(["decode", "decode", "verify", "chunk", "prompts"])
    # at most the positions of a listed case: 64 sequences of 4096 of 8 heads of 128 dims
    if shape in ("decode", "verify"):
        seqs = _log(rng, 1, 256 if shape == "decode" else 32)
        hi = min(32767, _log(rng, 30, 260000 // seqs))
        n = 1 if shape == "decode" else rng.randint(2, 16)
        return _attn(window, cap, seqs, heads, kv_heads, d, cache, page, deal, least=1 if n == 1 else 2, most=n, hi=hi)
    if shape == "chunk":
        return _attn(window, cap, _log(rng, 1, 32), heads, kv_heads, d, cache, page, deal, first=_log(rng, 17, 512), hi=_log(rng, 100, 5000))
    return _attn(window, cap, rng.randint(1, 4), heads, kv_heads, d, cache, page, deal, least=1, most=_log(rng, 17, 1100), hi=rng.choice([0, 200]))


def _dealt(case):
    """(pos, rows) of each sequence."""
    r, got = random.Random(case["deal"]), []
    for s in range(case["seqs"]):
        n = case["first"] if case["first"] and s == 0 else r.randint(case["least"], case["most"])
        got.append((r.randint(case["lo"], case["hi"]), n))
    return got


# ------------------------------------------------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _unit(g, shape):
    x = torch.randn(shape, generator=g, device="cuda")
    return x / x.norm(dim=-1, keepdim=True)


def _rows_inputs(case, g):
    """An append's q, k, v and the scale of its queries."""
    n, d = sum(m for _, m in _dealt(case)), case["d"]
    k, v = (torch.randn((n, case["kv_heads"], d), generator=g, device="cuda") for _ in range(2))
    q = torch.randn((n, case["heads"], d), generator=g, device="cuda")
    scale = 0.5 + torch.rand(case["heads"] * d, generator=g, device="cuda")
    t = torch.float32 if case["x"] == "f32" else torch.bfloat16
    return q.to(t), k.to(t), v.to(t), scale


def _held_inputs(case, g):
    """The rows that the pages hold, those of all sequences one behind another, in FP32."""
    shape = (sum(p + n for p, n in _dealt(case)), case["kv_heads"], case["d"])
    return _unit(g, shape), torch.randn(shape, generator=g, device="cuda")


def _attn_inputs(case, g):
    k, v = _held_inputs(case, g)
    n, d = sum(m for _, m in _dealt(case)), case["d"]
    spread = 6.0 if case["cap"] else 1.0
    q = _unit(g, (n, case["heads"], d)) * (d * spread) * (0.5 + torch.rand((1, case["heads"], d), generator=g, device="cuda"))
    return k, v, q.bfloat16()


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class _State:
    """What one program holds; its device cache goes with it."""
    cache = None

    def __del__(self):
        if self.cache is not None:
            self.cache.destroy()


def _tables(s, case, g):
    """The sequences' tables: positions, first rows, and pages in no order out of a pool with some to spare."""
    dealt, size = _dealt(case), case["page"]
    need = [(p + n + size - 1) // size for p, n in dealt]
    s.n_pages, s.max_pages = sum(need) + sum(need) // 8 + 1, max(need)
    order, table, at = torch.randperm(s.n_pages, generator=g, device="cuda").int(), [], 0
    for m in need:
        table.append(list(range(at, at + m)) + [0] * (s.max_pages - m))
        at += m
    s.pages = order[_ints(table).long()].contiguous()
    s.pos = _ints([p for p, _ in dealt])
    starts = [0]
    for _, n in dealt:
        starts.append(starts[-1] + n)
    s.n_rows, s.one_each = starts[-1], all(n == 1 for _, n in dealt)
    s.starts = _ints(starts)


# ---------------------------------------------------------------------------------------------- the framework's side

_backend = []


def _package():
    """The package under the name its own modules use, from the tree that is the working folder."""
    if "xtier_go_amd" not in sys.modules:
        if os.getcwd() not in sys.path:
            sys.path.insert(0, os.getcwd())
        sys.modules["xtier_go_amd"] = importlib.import_module("xtier-go_amd")
    return sys.modules["xtier_go_amd"]


def _hip():
    """The one backend (device and stream) that a program keeps open."""
    if not _backend:
        _backend.append(_package().HipBackend(0))
    return _backend[0]


def prepare(case, seed):
    s, g = _State(), _gen(seed)
    s.case = case
    kv, d = case["kv_heads"], case["d"]
    _tables(s, case, g)
    held = None
    if case["kind"] == "append":
        s.q, s.k, s.v, s.scale = _rows_inputs(case, g)
        s.q2 = torch.zeros_like(s.q)
    elif case["kind"] == "read":
        held = _held_inputs(case, g)
    else:
        *held, s.q = _attn_inputs(case, g)
        s.out = torch.zeros_like(s.q)
    s.k2, s.v2 = (torch.zeros((s.n_rows, kv, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    if own:
        pkg, s.b = _package(), _hip()
        dtype = {"nvfp4": pkg.KV_NVFP4, "fp8": pkg.KV_FP8, "bf16": pkg.KV_BF16}[case["cache"]]
        s.cache = s.b.paged_cache(kv, d, s.n_pages, case["page"], dtype)
        s.rows = s.b.paged_rows(s.pos, s.pages, s.n_rows, None if s.one_each else s.starts)
        if held is not None:
            starts = [0]
            for p, n in _dealt(case):
                starts.append(starts[-1] + p + n)
            torch.cuda.synchronize()
            whole = s.b.paged_rows(torch.zeros_like(s.pos), s.pages, starts[-1], _ints(starts))
            torch.cuda.synchronize()
            s.cache.append(whole, held[0], held[1], pkg.X_F32)
            s.b.finish()
    else:
        _plain_prepare(s, case, held)
    torch.cuda.synchronize()
    return s


def run(s):
    case = s.case
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attn": _plain_attention}[case["kind"]](s)
    pkg = _package()
    if case["kind"] == "attn":
        s.cache.attention(s.rows, s.q, s.out, case["heads"], pkg.X_BF16, case["window"], None, case["cap"])
        return s.out
    if case["kind"] == "append":
        x = pkg.X_F32 if case["x"] == "f32" else pkg.X_BF16
        s.cache.append(s.rows, s.k, s.v, x, s.q, s.q2, case["heads"], case["theta"], case["norm"], s.scale if case["norm"] else None)
        s.cache.read(s.rows, s.k2, s.v2, pkg.X_BF16)
        return s.q2, s.k2, s.v2
    s.cache.read(s.rows, s.k2, s.v2, pkg.X_BF16)
    return s.k2, s.v2


# ----------------------------------------------------------------------------------------------------- plain forms


_known = {}


def _steps(device):
    """Kept for a device: the values of the E4M3 codes 0 .. 126, the amax where a block's scale goes from each of them
    to the next, and the values of the E2M1 codes."""
    if device not in _known:
        c = torch.arange(127, device=device)
        e, m = c >> 3, (c & 7).double()
        steps = torch.where(e > 0, (1 + m / 8) * torch.exp2((e - 7).double()), m * 2.0 ** -9)
        mids = (steps[1:] + steps[:-1]) / 2 * 6   # exact; a tie goes to the even code
        mids = torch.where(c[:-1] % 2 == 1, torch.nextafter(mids, torch.zeros_like(mids)), mids)
        _known[device] = steps.float(), mids, torch.tensor(E2M1 + tuple(-v for v in E2M1), device=device)
    return _known[device]


def _encode(x, cache):
    """FP32 rows [n][kv][d] as the arrays that a pool holds of them."""
    if cache == "bf16":
        return (x.bfloat16(),)
    if cache == "fp8":
        amax = x.abs().amax(dim=-1, keepdim=True)
        s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
        return (x * (1.0 / s)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), s
    b = x.reshape(*x.shape[:-1], -1, 16)
    a = b.abs()
    amax = a.amax(dim=-1)
    steps, mids, _ = _steps(x.device)
    code = torch.maximum(torch.bucketize(amax.double(), mids), amax > 0)
    s = steps[code][..., None]
    e = ((a > 0.25 * s).to(torch.uint8) + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s) + (a > 2.5 * s) +
         (a >= 3.5 * s) + (a > 5.0 * s))   # products of at most 7 bits: exact
    e = torch.where(a > 0, e + (b < 0) * 8, 0).to(torch.uint8).reshape(*x.shape[:-1], -1, 2)
    return e[..., 0] | e[..., 1] << 4, code.to(torch.uint8)


def _decode(held, cache):
    """The values of such arrays, in FP32."""
    if cache == "bf16":
        return held[0].float()
    if cache == "fp8":
        return held[0].view(torch.float8_e4m3fn).float() * held[1]
    codes, scales = held
    steps, _, t = _steps(codes.device)
    v = torch.stack((t[(codes & 15).long()], t[(codes >> 4).long()]), dim=-1)
    return (v.reshape(*scales.shape, 16) * steps[scales.long()][..., None]).reshape(*scales.shape[:-1], -1)


def _plain_prepare(s, case, held):
    """The pool in its plain form: arrays [page][position in it][KV head][..]. The plan: each row's sequence, and the
    sequences of one row and of more, each kind as one padded batch."""
    kv, d, size, dealt = case["kv_heads"], case["d"], case["page"], _dealt(case)
    like = _encode(torch.zeros((1, kv, d), device="cuda"), case["cache"])
    s.kp, s.vp = (tuple(torch.zeros((s.n_pages, size, *a.shape[1:]), dtype=a.dtype, device="cuda") for a in like) for _ in range(2))
    s.seq = _ints([i for i, (_, n) in enumerate(dealt) for _ in range(n)]).long()
    if held is not None:
        at = 0
        for i, (p, n) in enumerate(dealt):
            where = torch.arange(p + n, device="cuda")
            page, slot = s.pages[i].long()[where // size], where % size
            for pool, rows in ((s.kp, held[0]), (s.vp, held[1])):
                for a, x in zip(pool, _encode(rows[at:at + p + n], case["cache"])):
                    a[page, slot] = x
            at += p + n
    s.groups = []
    for several in (False, True):
        which = [i for i, (_, n) in enumerate(dealt) if (n > 1) == several]
        if case["kind"] != "attn" or not which:
            continue
        lows = [max(0, dealt[i][0] - case["window"] + 1) if case["window"] else 0 for i in which]
        most, keys = max(dealt[i][1] for i in which), max(dealt[i][0] + dealt[i][1] - lo for i, lo in zip(which, lows))
        first = s.starts.tolist()
        into = _ints([first[i] + r for i in which for r in range(dealt[i][1])]).long()
        out_of = _ints([j * most + r for j, i in enumerate(which) for r in range(dealt[i][1])]).long()
        s.groups.append((_ints(which).long(), most, keys, into, out_of))


def _row_places(s):
    """Each row's position, its page and its place there."""
    at = s.pos[s.seq].long() + torch.arange(s.n_rows, device=s.pos.device) - s.starts[s.seq].long()
    return at, s.pages[s.seq, at // s.case["page"]].long(), at % s.case["page"]


def _rotated(x, at, theta):
    x = x.float()
    if theta == 0:
        return x
    half = x.shape[-1] // 2
    f = theta ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    angle = at.double()[:, None, None] * f
    c, sn = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * c - b * sn, b * c + a * sn), dim=-1)


def _normed(x):
    return x * (1.0 / torch.sqrt((x * x).sum(dim=-1, keepdim=True) + 1e-6))


def _plain_append(s):
    case = s.case
    at, page, slot = _row_places(s)
    q, k = _rotated(s.q, at, case["theta"]), _rotated(s.k, at, case["theta"])
    if case["norm"]:
        q, k = _normed(q) * s.scale.reshape(case["heads"], case["d"]), _normed(k)
    place = (page, slot)
    [a.index_put_(place, x) for a, x in zip(s.kp + s.vp, _encode(k, case["cache"]) + _encode(s.v.float(), case["cache"]))]
    return (q.to(s.q.dtype), *_plain_read(s))


def _plain_read(s):
    _, page, slot = _row_places(s)
    return tuple(_decode([a[page, slot] for a in pool], s.case["cache"]).bfloat16() for pool in (s.kp, s.vp))


def _plain_attention(s):
    out = torch.empty_like(s.q)
    [_plain_group(s, out, *group) for group in s.groups]
    return out


def _plain_group(s, out, which, most, keys, into, out_of):
    case = s.case
    heads, kv, d, size = case["heads"], case["kv_heads"], case["d"], case["page"]
    group, n, dev = heads // kv, which.numel(), out.device
    pos, rows = s.pos[which].long()[:, None], (s.starts[1:] - s.starts[:-1])[which].long()[:, None]
    lo = (pos - case["window"] + 1).clamp(min=0) if case["window"] else torch.zeros_like(pos)
    at = lo + torch.arange(keys, device=dev)                                                     # [seqs][keys]
    end = pos + rows
    page = torch.gather(s.pages[which].long(), 1, torch.minimum(at, end - 1) // size)
    k = _decode([a[page, at % size] for a in s.kp], case["cache"])                               # [seqs][keys][kv][d]
    v = _decode([a[page, at % size] for a in s.vp], case["cache"])
    k = k.permute(0, 2, 3, 1).contiguous()                                                       # [seqs][kv][d][keys]
    v = v.permute(0, 2, 1, 3).contiguous()                                                       # [seqs][kv][keys][d]
    q = torch.zeros((n * most, heads, d), device=dev)
    q[out_of] = s.q[into].float()
    q = q.reshape(n, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, d).contiguous()
    score = torch.matmul(q, k) * (1.0 / math.sqrt(d))
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    t = (pos + torch.arange(most, device=dev))[:, :, None]                                       # [seqs][rows][1]
    hide = (at[:, None] > t) | (at >= end)[:, None]
    if case["window"]:
        hide = hide | (t - at[:, None] >= case["window"])
    score = score.reshape(n, kv, group, most, keys).masked_fill(hide[:, None, None], -math.inf)
    w = torch.exp(score - score.amax(dim=-1, keepdim=True))
    y = torch.matmul(w.reshape(n, kv, group * most, keys), v).reshape(n, kv, group, most, d) / w.sum(dim=-1, keepdim=True)
    out[into] = y.permute(0, 3, 1, 2, 4).reshape(n * most, heads, d)[out_of].to(out.dtype)


# ---------------------------------------------------------------------------------------------------- what is needed


def _row_bytes(case):
    """Bytes that one position's keys and values take in a page."""
    d = case["d"]
    return 2 * case["kv_heads"] * {"nvfp4": d // 2 + d // 16, "fp8": d + 4, "bf16": 2 * d}[case["cache"]]


def work(case):
    dealt, d, heads, kv = _dealt(case), case["d"], case["heads"], case["kv_heads"]
    n = sum(m for _, m in dealt)
    back = n * (_row_bytes(case) + 2 * kv * d * 2)
    if case["kind"] == "read":
        return {"bytes": back, "flops": 0}
    if case["kind"] == "append":   # q in and out, k and v in, their pages written, and read back
        size = 4 if case["x"] == "f32" else 2
        return {"bytes": n * (2 * heads + 2 * kv) * d * size + n * _row_bytes(case) + back, "flops": 0}
    keys = pairs = 0
    for p, m in dealt:
        w = case["window"] or p + m
        keys += p + m - max(0, p - w + 1)
        pairs += sum(min(t + 1, w) for t in range(p, p + m))
    return {"bytes": keys * _row_bytes(case) + 2 * n * heads * d * 2, "flops": 4 * d * heads * pairs}


# ------------------------------------------------------------------------------------------------------ in 64 bits


def _nearest(y, bits, low):
    """y >= 0 to the nearest value of `bits` significant bits and a step of at least `low`, ties to even."""
    _, e = torch.frexp(y)
    step = torch.exp2((e - bits).double()).clamp(min=low)
    return torch.round(y / step) * step


def _stored(x, cache):
    """The values that a pool of this type holds of rows."""
    x = x.double()
    if cache == "bf16":
        return x.bfloat16().double()
    if cache == "fp8":   # the scale and its inverse, and the products that are rounded to codes, are FP32 numbers
        x = x.float()
        amax = x.abs().amax(dim=-1, keepdim=True)
        s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
        y = (x * (1.0 / s)).double()
        return _nearest(y.abs(), 4, 2.0 ** -9).clamp(max=448) * y.sign() * s.double()
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    amax = b.abs().amax(dim=-1, keepdim=True)
    s = _nearest(amax / 6, 4, 2.0 ** -9).clamp(max=448)
    s = torch.where(amax > 0, s.clamp(min=2.0 ** -9), torch.ones_like(s))
    return (_nearest(b.abs() / s, 2, 0.5).clamp(max=6) * s * b.sign()).reshape(x.shape)


def exact(case, seed):
    g, s, dealt, cache = _gen(seed), _State(), _dealt(case), case["cache"]
    _tables(s, case, g)   # (draws the pages' order first, as prepare does)
    heads, kv, d = case["heads"], case["kv_heads"], case["d"]
    if case["kind"] == "append":
        q, k, v, scale = _rows_inputs(case, g)
        q, k = q.double(), k.double()
        if case["theta"]:
            at = torch.tensor([p + r for p, n in dealt for r in range(n)], dtype=torch.float64, device=q.device)
            turn = at[:, None, None] * case["theta"] ** (-2.0 * torch.arange(d // 2, dtype=torch.float64, device=q.device) / d)
            turn = torch.polar(torch.ones_like(turn), turn)
            q, k = (torch.view_as_real(torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * turn)
                    .transpose(-1, -2).reshape(x.shape) for x in (q, k))
        if case["norm"]:
            q, k = (x / ((x ** 2).sum(dim=-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
            q = q * scale.double().reshape(heads, d)
        return q, _stored(k, cache), _stored(v, cache)
    if case["kind"] == "read":
        k, v = _held_inputs(case, g)
        keep, at = [], 0
        for p, n in dealt:
            keep += range(at + p, at + p + n)
            at += p + n
        return tuple(_stored(x[torch.tensor(keep, device=x.device)], cache) for x in (k, v))
    k, v, q = _attn_inputs(case, g)
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    at = row = 0
    for p, n in dealt:
        lo = max(0, p - case["window"] + 1) if case["window"] else 0
        kk, vv = (_stored(x[at + lo:at + p + n], cache).transpose(0, 1).contiguous() for x in (k, v))   # [kv][keys][d]
        key = torch.arange(lo, p + n, device=q.device)[None]
        for r in range(0, n, 256):
            m = min(256, n - r)
            t = torch.arange(p + r, p + r + m, device=q.device)[:, None]
            seen = key <= t
            if case["window"]:
                seen = seen & (key > t - case["window"])
            x = q[row + r:row + r + m].double().reshape(m, kv, heads // kv, d).permute(1, 2, 0, 3).reshape(kv, -1, d)
            z = torch.bmm(x, kk.transpose(1, 2).contiguous()) / math.sqrt(d)
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            z = torch.where(seen, z.reshape(kv, heads // kv, m, -1), -math.inf).softmax(dim=-1)
            y = torch.bmm(z.reshape(kv, (heads // kv) * m, -1), vv)
            out[row + r:row + r + m] = y.reshape(kv, heads // kv, m, d).permute(2, 0, 1, 3).reshape(m, heads, d)
        at, row = at + p + n, row + n
    return out
