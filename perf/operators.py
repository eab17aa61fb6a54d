"""Performance cases of the 4-bit KV cache and of attention with capped, biased and masked scores.

The operators: the rows of a call quantised into an NVFP4 cache as they are written, and read back
(xtg_hip_kv_write, xtg_hip_kv_read); attention over that cache, and attention over any cache (NVFP4, FP8 or BF16) or
over the call's own keys alone whose scores are capped by a tanh, biased by distance, or masked by document, prefix and
window (xtg_hip_attention_ext).

The NVFP4 cache holds, for each (position, KV head) and 16 dims, an E4M3 scale s = the nearest of amax / 6 (ties to
even, at most 448, at least 2^-9 unless the block is zero) and E2M1 codes of x / s (nearest, ties to even, at most 6).
A row at position t sees the keys at positions first <= p < end, where end is t + 1 unless it is given, and
p > t - window when there is a window. Its scores are q.k * scale, then cap * tanh(score / cap), then -slope * |t - p|.

Head layouts, rings, windows and contexts are those of the two configurations of xtier-go_amd/workloads.py and of its
tests. Rows are BF16: keys are unit vectors, and queries are scaled so that a row's scores spread over several units.
"""
import importlib
import math
import os
import sys

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _attn(cache, n_q, ctx, heads, kv_heads, d, ring=0, window=0, cap=0.0, alibi=False, docs="", prefix=0):
    return {"kind": "attn", "cache": cache, "n_q": n_q, "ctx": ctx, "heads": heads, "kv_heads": kv_heads, "d": d,
            "ring": ring, "window": window, "cap": cap, "alibi": alibi, "docs": docs, "prefix": prefix}


def listed():
    return [
        # one decoded token's key and value rows of one layer, as FP32 projections leave them
        {"name": "kv-1row", "kind": "kv", "n": 1, "pos": 4095, "kv_heads": 8, "d": 128, "ring": 0, "x": "f32"},
        # a prompt chunk that runs over the end of a sliding layer's ring
        {"name": "kv-500rows-ring", "kind": "kv", "n": 500, "pos": 1900, "kv_heads": 4, "d": 256, "ring": 1040,
         "x": "f32"},
        # a whole long context moved into a cache (a prefix shared between sessions), an odd number of rows
        {"name": "kv-32749rows", "kind": "kv", "n": 32749, "pos": 13, "kv_heads": 8, "d": 128, "ring": 0, "x": "bf16"},
        # one token over a long 4-bit cache: a global layer of the 4B-shaped configuration
        dict(_attn("nvfp4", 1, 32768, 32, 8, 128), name="attn4-1row-32k"),
        # a speculative verify step over a full 4-bit ring: a sliding layer of the real configuration
        dict(_attn("nvfp4", 8, 5000, 16, 4, 256, ring=1040, window=1024), name="attn4-8rows-ring"),
        # the ragged tail of a prompt, heads of 64 dims
        dict(_attn("nvfp4", 37, 5001, 16, 8, 64), name="attn4-37rows-5k"),
        # a prompt chunk in the middle of a long prompt
        dict(_attn("nvfp4", 512, 16384, 32, 8, 128), name="attn4-512rows-16k"),
        # one token with capped scores over a BF16 cache
        dict(_attn("bf16", 1, 8191, 16, 4, 256, cap=50.0), name="capped-1row-8k"),
        # a short turn with a distance bias over an FP8 cache
        dict(_attn("fp8", 45, 4000, 32, 8, 128, alibi=True), name="alibi-45rows-4k"),
        # documents packed into one sequence, no cache
        dict(_attn("none", 2047, 0, 32, 8, 128, docs="700+1+299+1047"), name="docs-2047rows"),
        # a sequence whose prefix is seen both ways, its start in a 4-bit cache, capped scores
        dict(_attn("nvfp4", 1500, 1000, 16, 4, 256, cap=30.0, prefix=1800), name="prefix-1500rows"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.3:
        kv_heads, d = rng.choice([(8, 128), (4, 256), (8, 64), (2, 128)])
        ring = rng.choice([0, 0, 1040, 1088])
        x = rng.choice(["f32", "bf16"])
        most = 32768 * 1024 // (kv_heads * d) // (2 if x == "f32" else 1) - 32
        return {"kind": "kv", "n": _log(rng, 1, ring if ring else min(32768, most)), "pos": rng.randint(0, 5000),
                "kv_heads": kv_heads, "d": d, "ring": ring, "x": x}
    heads, kv_heads, d = rng.choice([(32, 8, 128), (16, 4, 256), (16, 8, 64), (32, 8, 128), (12, 4, 128)])
    n_q = rng.choice([1, _log(rng, 2, 16), _log(rng, 17, 2048), _log(rng, 17, 2048)])
    cache = rng.choice(["nvfp4", "nvfp4", "nvfp4", "fp8", "bf16", "none"])
    if cache == "none":
        n_q = max(n_q, 17)
        ctx = 0
    else:   # at most the products of 512 rows of 32 heads of 128 after 16384 positions
        ctx = _log(rng, 100, min(32768, max(200, 4096 * 512 * 16384 // (n_q * heads * d) - n_q)))
    c = _attn(cache, n_q, ctx, heads, kv_heads, d)
    kinds = ["cap", "alibi", "docs", "prefix", "window"]
    kind = rng.choice(kinds + ["none"] * 5 if cache == "nvfp4" else kinds)
    if cache != "none" and rng.random() < 0.25:
        c["ring"], c["window"] = (1040 if d == 256 else 1088), 1024
    if kind == "cap":
        c["cap"] = float(rng.choice([15, 30, 50]))
    if kind == "alibi":
        c["alibi"] = True
    if kind == "window":
        c["window"] = rng.choice([256, 1024])
    if kind == "docs":   # the first document began before the call where there is a cache
        cuts = sorted(rng.randint(0, n_q) for _ in range(rng.randint(1, 6)))
        c["docs"] = "+".join(str(b - a) for a, b in zip([0] + cuts, cuts + [n_q]) if b > a)
    if kind == "prefix":
        c["prefix"] = ctx + rng.randint(1, n_q)
    return c


# ------------------------------------------------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _unit(g, shape):
    x = torch.randn(shape, generator=g, device="cuda")
    return x / x.norm(dim=-1, keepdim=True)


def _kv_inputs(case, seed):
    g = _gen(seed)
    shape = (case["n"], case["kv_heads"], case["d"])
    k, v = _unit(g, shape), torch.randn(shape, generator=g, device="cuda")
    return (k.bfloat16(), v.bfloat16()) if case["x"] == "bf16" else (k, v)


def _held(case):
    """The first position that the cache still holds, and how many it holds."""
    n = min(case["ctx"], case["ring"]) if case["ring"] else case["ctx"]
    return case["ctx"] - n, n


def _attn_inputs(case, seed):
    """The cached rows in FP32 [held][kv][d], and the call's q, k, v in BF16."""
    g = _gen(seed)
    n, held, d = case["n_q"], _held(case)[1], case["d"]
    shape = (held, case["kv_heads"], d)
    kc, vc = _unit(g, shape), torch.randn(shape, generator=g, device="cuda")
    spread = 6.0 if case["cap"] else 1.0
    q = _unit(g, (n, case["heads"], d)) * (d * spread) * (0.5 + torch.rand((1, case["heads"], d), generator=g,
                                                                          device="cuda"))
    k = _unit(g, (n, case["kv_heads"], d))
    v = torch.randn((n, case["kv_heads"], d), generator=g, device="cuda")
    return kc, vc, q.bfloat16(), k.bfloat16(), v.bfloat16()


def _spans(case):
    """(first, end) of each row of the call as lists, or None where the case does not give them."""
    n, ctx = case["n_q"], case["ctx"]
    first = end = None
    if case["docs"]:
        first, at = [], 0
        for length in map(int, case["docs"].split("+")):
            first += [ctx + at if at else 0] * length
            at += length
    if case["prefix"]:
        end = [max(ctx + i + 1, case["prefix"]) for i in range(n)]
    return first, end


def _slopes(case):
    return [2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])] if case["alibi"] else None


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


class _State:
    """What one program holds; its device cache goes with it."""
    cache = None

    def __del__(self):
        if self.cache is not None:
            self.cache.destroy()


def prepare(case, seed):
    s = _State()
    s.case = case
    if case["kind"] == "kv":
        s.k, s.v = _kv_inputs(case, seed)
        kept = min(case["n"], case["ring"]) if case["ring"] else case["n"]
        s.read = (case["pos"] + case["n"] - kept, kept)
        s.k2, s.v2 = torch.zeros_like(s.k[:kept]), torch.zeros_like(s.v[:kept])
        if own:
            s.b, s.x = _hip(), _package().X_BF16 if case["x"] == "bf16" else _package().X_F32
            s.cache = s.b.kv_cache(case["kv_heads"], case["d"], case["pos"] + case["n"], case["ring"],
                                   _package().KV_NVFP4)
        torch.cuda.synchronize()
        return s
    kc, vc, s.q, s.k, s.v = _attn_inputs(case, seed)
    first, end = _spans(case)
    s.first = torch.tensor(first, dtype=torch.int32, device="cuda") if first else None
    s.end = torch.tensor(end, dtype=torch.int32, device="cuda") if end else None
    s.slopes = torch.tensor(_slopes(case), device="cuda") if case["alibi"] else None
    s.out = torch.zeros_like(s.q)
    p0, held = _held(case)
    if own:
        pkg, s.b = _package(), _hip()
        torch.cuda.synchronize()
        if held:
            dtype = {"nvfp4": pkg.KV_NVFP4, "fp8": pkg.KV_FP8, "bf16": pkg.KV_BF16}[case["cache"]]
            s.cache = s.b.kv_cache(case["kv_heads"], case["d"], case["ctx"], case["ring"], dtype)
            s.cache.write(p0, held, kc, vc, pkg.X_F32)
            s.b.finish()
    elif case["cache"] == "nvfp4":
        s.kc, s.vc = _quantise(kc), _quantise(vc)
    elif case["cache"] == "fp8":
        s.kc, s.vc = _fp8(kc), _fp8(vc)
    else:
        s.kc, s.vc = kc.bfloat16(), vc.bfloat16()
    torch.cuda.synchronize()
    return s


def run(s):
    case = s.case
    if case["kind"] == "kv":
        if not own:
            return _dequantise(*_quantise(s.k)).to(s.k.dtype)[-s.read[1]:], \
                _dequantise(*_quantise(s.v)).to(s.v.dtype)[-s.read[1]:]
        s.cache.write(case["pos"], case["n"], s.k, s.v, s.x)
        s.cache.read(s.read[0], s.read[1], s.k2, s.v2, s.x)
        return s.k2, s.v2
    if not own:
        return _plain_attention(s)
    s.b.attention_ext(s.cache, s.q, s.k, s.v, s.out, case["n_q"], case["ctx"], case["heads"], case["kv_heads"],
                      case["d"], _package().X_BF16, case["window"], None, case["cap"], s.slopes, s.first, s.end)
    return s.out


# ----------------------------------------------------------------------------------------------------- plain forms


_tables = {}


def _table(device):
    """Kept for a device: the values of the E4M3 codes 0 .. 126, the amax where a block's scale goes from each of them
    to the next, and the values of the E2M1 codes."""
    if device not in _tables:
        c = torch.arange(127, device=device)
        e, m = c >> 3, (c & 7).double()
        steps = torch.where(e > 0, (1 + m / 8) * torch.exp2((e - 7).double()), m * 2.0 ** -9)
        mids = (steps[1:] + steps[:-1]) / 2 * 6   # exact; a tie goes to the even code
        mids = torch.where(c[:-1] % 2 == 1, torch.nextafter(mids, torch.zeros_like(mids)), mids)
        _tables[device] = steps.float(), mids, torch.tensor(E2M1 + tuple(-v for v in E2M1), device=device)
    return _tables[device]


def _quantise(x):
    """Rows [n][heads][d] as E2M1 codes, two to a byte [n][heads][d / 2], and E4M3 scale codes [n][heads][d / 16]."""
    b = x.float().reshape(*x.shape[:-1], -1, 16)
    a = b.abs()
    amax = a.amax(dim=-1)
    steps, mids, _ = _table(x.device)
    code = torch.maximum(torch.bucketize(amax.double(), mids), amax > 0)
    s = steps[code][..., None]
    e = ((a > 0.25 * s).to(torch.uint8) + (a >= 0.75 * s) + (a > 1.25 * s) + (a >= 1.75 * s) + (a > 2.5 * s) +
         (a >= 3.5 * s) + (a > 5.0 * s))   # products of at most 7 bits: exact
    e = torch.where(a > 0, e + (b < 0) * 8, 0).to(torch.uint8).reshape(*x.shape[:-1], -1, 2)
    return e[..., 0] | e[..., 1] << 4, code.to(torch.uint8)


def _dequantise(codes, scales):
    steps, _, t = _table(codes.device)
    v = torch.stack((t[(codes & 15).long()], t[(codes >> 4).long()]), dim=-1)
    return (v.reshape(*scales.shape, 16) * steps[scales.long()][..., None]).reshape(*scales.shape[:-1], -1)


def _fp8(x):
    """E4M3 codes and a scale amax / 448 for each (row, head)."""
    amax = x.abs().amax(dim=-1, keepdim=True)
    s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    return (x * (1.0 / s)).clamp(-448, 448).to(torch.float8_e4m3fn), s


def _plain_attention(s):
    case = s.case
    n, ctx, heads, kv, d = case["n_q"], case["ctx"], case["heads"], case["kv_heads"], case["d"]
    if case["cache"] == "nvfp4":
        kc, vc = _dequantise(*s.kc), _dequantise(*s.vc)
    elif case["cache"] == "fp8":
        kc, vc = s.kc[0].float() * s.kc[1], s.vc[0].float() * s.vc[1]
    else:
        kc, vc = s.kc.float(), s.vc.float()
    k = torch.cat((kc, s.k.float())).permute(1, 2, 0)[:, None].contiguous()                       # [kv][1][d][keys]
    v = torch.cat((vc, s.v.float())).permute(1, 0, 2)[:, None].contiguous()                       # [kv][1][keys][d]
    q = s.q.float().reshape(n, kv, heads // kv, d).permute(1, 2, 0, 3).contiguous()               # [kv][group][n][d]
    score = torch.matmul(q, k) * (1.0 / math.sqrt(d))
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    p0 = _held(case)[0]
    at = torch.arange(p0, ctx + n, device=q.device)
    t = torch.arange(ctx, ctx + n, device=q.device)[:, None]
    if s.slopes is not None:
        score = score - s.slopes.reshape(kv, heads // kv, 1, 1) * (t - at).abs()
    hide = at >= (t + 1 if s.end is None else s.end[:, None])
    if s.first is not None:
        hide = hide | (at < s.first[:, None])
    if case["window"]:
        hide = hide | (t - at >= case["window"])
    score = score.masked_fill(hide, -math.inf)
    w = torch.exp(score - score.amax(dim=-1, keepdim=True))
    out = torch.matmul(w, v) / w.sum(dim=-1, keepdim=True)
    return out.permute(2, 0, 1, 3).reshape(n, heads, d).to(s.q.dtype)


# ---------------------------------------------------------------------------------------------------- what is needed


def _row_bytes(case):
    """Bytes that one cached position's keys and values take."""
    d = case["d"]
    return 2 * case["kv_heads"] * {"nvfp4": d // 2 + d // 16, "fp8": d + 4, "bf16": 2 * d, "none": 0}[case["cache"]]


def work(case):
    if case["kind"] == "kv":   # written: rows in, codes and scales out; read back: the other way round
        n = case["n"] * case["kv_heads"] * case["d"] * 2
        kept = min(case["n"], case["ring"] or case["n"]) * case["kv_heads"] * case["d"] * 2
        size = 4 if case["x"] == "f32" else 2
        return {"bytes": kept * size * 2 + 2 * (kept // 2 + kept // 16), "flops": 0}
    n, ctx, heads, kv, d = case["n_q"], case["ctx"], case["heads"], case["kv_heads"], case["d"]
    first, end = _spans(case)
    p0, pairs, lowest = _held(case)[0], 0, ctx
    for i in range(n):
        lo = max(p0, first[i] if first else 0, ctx + i + 1 - case["window"] if case["window"] else 0)
        pairs += max(0, (end[i] if end else ctx + i + 1) - lo)
        lowest = min(lowest, lo)
    return {"bytes": (ctx - lowest) * _row_bytes(case) + 2 * n * d * (2 * heads + 2 * kv), "flops": 4 * d * heads * pairs}


# ------------------------------------------------------------------------------------------------------ in 64 bits


def _nearest(y, bits, low):
    """y >= 0 to the nearest value of `bits` significant bits and a step of at least `low`, ties to even."""
    _, e = torch.frexp(y)
    step = torch.exp2((e - bits).double()).clamp(min=low)
    return torch.round(y / step) * step


def _stored_nvfp4(x):
    b = x.double().reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    amax = b.abs().amax(dim=-1, keepdim=True)
    s = _nearest(amax / 6, 4, 2.0 ** -9).clamp(max=448)
    s = torch.where(amax > 0, s.clamp(min=2.0 ** -9), torch.ones_like(s))
    return (_nearest(b.abs() / s, 2, 0.5).clamp(max=6) * s * b.sign()).reshape(x.shape)


def _stored_fp8(x):
    amax = x.abs().amax(dim=-1, keepdim=True)
    s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
    y = (x * (1.0 / s)).double()
    return _nearest(y.abs(), 4, 2.0 ** -9).clamp(max=448) * y.sign() * s.double()


def exact(case, seed):
    if case["kind"] == "kv":
        kept = min(case["n"], case["ring"]) if case["ring"] else case["n"]
        k, v = _kv_inputs(case, seed)
        return _stored_nvfp4(k[-kept:]), _stored_nvfp4(v[-kept:])
    kc, vc, q, k, v = _attn_inputs(case, seed)
    stored = {"nvfp4": _stored_nvfp4, "fp8": _stored_fp8, "bf16": lambda x: x.bfloat16().double(),
              "none": lambda x: x.double()}[case["cache"]]
    n, ctx, group = case["n_q"], case["ctx"], case["heads"] // case["kv_heads"]
    kk, vv = torch.cat((stored(kc), k.double())), torch.cat((stored(vc), v.double()))
    first, end = _spans(case)
    slopes, out = _slopes(case), torch.empty(q.shape, dtype=torch.float64, device=q.device)
    p0 = ctx - _held(case)[1]
    key = torch.arange(p0, ctx + n, device=q.device, dtype=torch.float64)[None, :]
    for r in range(0, n, 256):   # rows r .. r + m
        m = min(256, n - r)
        t = torch.arange(ctx + r, ctx + r + m, device=q.device, dtype=torch.float64)[:, None]
        lo = torch.zeros_like(t) if first is None else torch.tensor(first[r:r + m], device=q.device).double()[:, None]
        if case["window"]:
            lo = torch.maximum(lo, t - case["window"] + 1)
        hi = t if end is None else torch.tensor(end[r:r + m], device=q.device).double()[:, None] - 1
        seen = (key >= lo) & (key <= hi)
        for h in range(case["heads"]):
            z = q[r:r + m, h].double() @ kk[:, h // group].T / math.sqrt(case["d"])
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            if slopes:
                z = z - slopes[h] * (t - key).abs()
            out[r:r + m, h] = torch.where(seen, z, -math.inf).softmax(dim=-1) @ vv[:, h // group]
    return out
