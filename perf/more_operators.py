"""Performance cases of the operators around a layer whose projections are 8-bit: the norms
between two blocks with the quantiser of the next product, the product of 8-bit codes,
and decode attention of a batch that shares a long prefix, each through its public entry
point (the C ABI of include/jllm_hip.h) or, where `own` is false, in its plain form.

Hidden sizes, projections and head layouts are those of the repository's decoder
configuration (2560 / 9728, 32 / 8 heads x 128), of its tests, and generic ones; `draw`
spreads over the ranges around them.

A case's "kind":
  norms    branch norm, gate, scaled residual, norm for the next block, codes (block_norms)
  gemm     product of 8-bit codes with a scale for each token and channel (gemm_i8)
  prefix   one query row of each of B sequences over a shared prefix and its own pages
           (flash_attention_decode_paged_prefix)
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6


def listed():
    return [
        # one user's decode step between attention and feed-forward: residual add and norm, where latency is all there is
        _norms("norms_one", rows=1, hidden=2560),
        # a batch's decode step, norms on both sides of the block, fp32 residual stream, codes for an 8-bit product
        _norms("norms_batch", rows=64, hidden=2560, post=True, wide=True, codes=True),
        # a prompt through a block with gated output and scaled branch, ragged row count
        _norms("norms_prompt", rows=8191, hidden=4096, post=True, gate="rows", act=1, branch=0.22),
        # one user's down projection: the weights are read once, little else
        _gemm("gemm_one", N=1, M=2560, K=9728),
        # a full batch's fused q / k / v projection
        _gemm("gemm_batch", N=64, M=6144, K=2560),
        # a prompt chunk's gate and up projections
        _gemm("gemm_prompt", N=2048, M=19456, K=2560),
        # ragged rows against an odd vocabulary: fp32 logits, biased, output rows not aligned
        _gemm("gemm_odd", N=251, M=32003, K=2064, f32=True, bias=True),
        # long prompts of several users through a wide layer: the largest product
        _gemm("gemm_large", N=8192, M=8192, K=8192),
        # a few chats under one system prompt
        _prefix("prefix_few", B=4, prefix=2048, ctx=200, int8=True),
        # a full batch of chats under one system prompt, two padded rows among them
        _prefix("prefix_chat", B=48, prefix=1500, ctx=1024, int8=True),
        # many questions about one long document: the largest
        _prefix("prefix_document", B=64, prefix=32768, ctx=512, page=32),
        # sliding-window layers, one KV head for twelve query heads, prefix and window end inside pages
        _prefix("prefix_window", B=17, prefix=5003, ctx=300, heads=12, kv=1, hd=96, page=64, window=4096),
    ]


def _norms(name, rows, hidden, post=False, gate="", act=0, branch=1.0, res=1.0, wide=False, codes=False):
    """gate: "" none, "one" a vector for all rows, "rows" one for each; act: 0 as it is,
    1 its sigmoid, 2 its tanh; wide: fp32 residual stream; codes: int8 codes for fp16 rows."""
    c = {"kind": "norms", "rows": rows, "hidden": hidden, "post": post, "gate": gate, "act": act, "branch": branch,
         "res": res, "wide": wide, "codes": codes}
    return dict(c, name=name) if name else c


def _gemm(name, N, M, K, f32=False, bias=False):
    c = {"kind": "gemm", "N": N, "M": M, "K": K, "f32": f32, "bias": bias}
    return dict(c, name=name) if name else c


def _prefix(name, B, prefix, ctx, heads=32, kv=8, hd=128, page=16, int8=False, window=0):
    c = {"kind": "prefix", "B": B, "prefix": prefix, "ctx": ctx, "heads": heads, "kv": kv, "hd": hd, "page": page,
         "int8": int8, "window": window}
    return dict(c, name=name) if name else c


def _logint(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["norms", "gemm", "gemm", "prefix", "prefix"])
    if kind == "norms":
        hidden = 8 * _logint(rng, 8, 2048)
        rows = _logint(rng, 1, min(8191, 8191 * 4096 // hidden))
        return _norms("", rows, hidden, rng.random() < 0.6, rng.choice(["", "", "one", "rows"]), rng.randint(0, 2),
                      rng.choice([1.0, 0.25 + rng.random()]), rng.choice([1.0, 0.25 + rng.random()]),
                      rng.random() < 0.4, rng.random() < 0.4)
    if kind == "gemm":
        K = 16 * _logint(rng, 1, 1024)
        M = _logint(rng, 16, min(65536, (1 << 27) // K))
        N = _logint(rng, 1, max(1, min(8192, (1 << 38) // (K * M))))
        return _gemm("", N, M, K, rng.random() < 0.4, rng.random() < 0.4)
    heads, kv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (16, 4, 128), (16, 2, 128), (8, 2, 64), (8, 8, 64),
                                (12, 1, 96), (4, 1, 32)])
    B = _logint(rng, 1, 96)
    # no more than the largest listed case in products, nor in what it reads
    prefix = _logint(rng, 1, min(65536, (1 << 33) // (B * heads * hd), 32768 * 1024 // (kv * hd)))
    ctx = _logint(rng, 1, min(2048, 50000 // B))
    return _prefix("", B, prefix, ctx, heads, kv, hd, rng.choice([16, 16, 32, 64, 256]), rng.random() < 0.5,
                   rng.choice([0, 0, 0, _logint(rng, 1, 8192)]))


# ---- inputs -----------------------------------------------------------------------

class State:
    pass


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _own_lengths(c):
    """Tokens of a batch's rows behind the prefix: the longest is `ctx`, every fourth has
    only begun, every 23rd row is padding (-1)."""
    r = random.Random("%d %d" % (c["B"], c["ctx"]))
    return [c["ctx"] if i == 0 else -1 if i % 23 == 22 else r.randint(0, min(3, c["ctx"])) if i % 4 == 3 else
            r.randint(1, c["ctx"]) for i in range(c["B"])]


def _pages(c, n):
    return (max(n, 0) + c["page"] - 1) // c["page"]


def prepare(case, seed):
    return {"norms": _prepare_norms, "gemm": _prepare_gemm, "prefix": _prepare_prefix}[case["kind"]](case, seed)


def _prepare_norms(c, seed):
    g, s = _gen(seed), State()
    s.c, s.kind = c, "norms"
    rows, hidden = c["rows"], c["hidden"]
    stream = torch.float32 if c["wide"] else torch.float16
    s.x = _randn(g, rows, hidden).half()
    # a residual stream has a few channels that are far larger than the others
    big = torch.where(torch.rand((hidden,), device=DEV, generator=g) < 0.01, 20.0, 1.0)
    s.residual = (_randn(g, rows, hidden) * 3 * big).to(stream)
    s.pre = 1 + 0.2 * _randn(g, hidden)
    s.post = 1 + 0.2 * _randn(g, hidden) if c["post"] else None
    s.gate = None
    if c["gate"]:
        s.gate = _randn(g, rows if c["gate"] == "rows" else 1, hidden).half()
    s.h = torch.zeros((rows, hidden), dtype=stream, device=DEV)
    if c["codes"]:
        s.codes = torch.zeros((rows, hidden), dtype=torch.int8, device=DEV)
        s.scales = torch.zeros((rows,), device=DEV)
        s.values = torch.zeros((rows, hidden), device=DEV)
    else:
        s.y = torch.zeros((rows, hidden), dtype=torch.float16, device=DEV)
    return s


def _codes(x):
    """Codes of a matrix with a scale for each row."""
    scale = x.abs().amax(-1, keepdim=True) / 127
    return torch.round(x / scale).to(torch.int8), scale[:, 0].contiguous()


def _prepare_gemm(c, seed):
    g, s = _gen(seed), State()
    s.c, s.kind = c, "gemm"
    s.x, s.xs = _codes(_randn(g, c["N"], c["K"]))
    s.w, s.ws = _codes(_randn(g, c["M"], c["K"]) / math.sqrt(c["K"]))
    s.bias = _randn(g, c["M"]) if c["bias"] else None
    s.out = torch.zeros((c["N"], c["M"]), dtype=torch.float32 if c["f32"] else torch.float16, device=DEV)
    return s


def _prepare_prefix(c, seed):
    g, s = _gen(seed), State()
    s.c, s.kind = c, "prefix"
    B, H, KV, hd, page = c["B"], c["heads"], c["kv"], c["hd"], c["page"]
    lens = _own_lengths(c)
    used = [_pages(c, n) for n in lens]
    shared = _pages(c, c["prefix"])
    s.n_pages = shared + sum(used) + 3
    s.prefix_len, s.lens = _ints([c["prefix"]]), _ints(lens)
    s.width = max(max(used), 1)
    # all pages lie anywhere in the pool; entries behind a sequence's last page are -1
    ids = torch.randperm(s.n_pages, device=DEV, generator=g).int()[:shared + sum(used)]
    s.prefix_table = ids[:shared].contiguous()
    at = torch.arange(s.width, device=DEV)[None] < _ints(used)[:, None]
    s.table = torch.full((B, s.width), -1, dtype=torch.int32, device=DEV)
    s.table[at] = ids[shared:]
    s.q = (_randn(g, B, H * hd) * 1.5).half()
    shape = (s.n_pages, page, KV, hd)
    s.ks = s.vs = None
    if c["int8"]:
        s.kp, s.vp = (torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=g) for _ in range(2))
        s.ks, s.vs = (torch.rand(shape[:3], device=DEV, generator=g) * 0.02 + 0.01 for _ in range(2))
    else:
        s.kp, s.vp = (torch.randn(shape, dtype=torch.float16, device=DEV, generator=g) for _ in range(2))
    s.scale = 1.0 / math.sqrt(hd)
    s.out = torch.zeros((B, H * hd), dtype=torch.float16, device=DEV)
    return s


# ---- one pass ---------------------------------------------------------------------

def run(s):
    if own:
        return {"norms": _own_norms, "gemm": _own_gemm, "prefix": _own_prefix}[s.kind](s)
    return {"norms": _plain_norms, "gemm": _plain_gemm, "prefix": _plain_prefix}[s.kind](s)


def _bound(s, name, *args):
    """A C-ABI call with its arguments converted once, as a program's binding keeps it."""
    if not hasattr(s, "call"):
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "genie-ai-runtime_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import jllm
        f = getattr(jllm.lib(), name)
        args = args[0](jllm.lib())
        conv = [None if a is None else t(a.data_ptr() if hasattr(a, "data_ptr") else a) for t, a in zip(f.argtypes, args)]
        conv.append(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        s.call = (f, conv, jllm.check)
    f, conv, check = s.call
    st = f(*conv)
    if st:
        check(st, name)


def _workspace(s, n):
    s.space = torch.empty((max(n, 16),), dtype=torch.uint8, device=DEV)
    return [s.space, s.space.numel()]


def _own_norms(s):
    c = s.c

    def args(lib):
        n = c["hidden"]
        codes = c["codes"]
        return [s.h, n, s.residual, n, int(c["wide"]), s.x, n, s.post, s.gate, n if c["gate"] == "rows" else 0,
                c["act"], c["branch"], c["res"], s.pre, 1, EPS, None if codes else s.y, n,
                s.codes if codes else None, n, s.scales if codes else None, c["rows"], n]

    _bound(s, "jllm_hip_block_norms", args)
    return _norms_outputs(s)


def _norms_outputs(s):
    if not s.c["codes"]:
        return [s.h, s.y]
    # codes as the values they stand for
    return [s.h, torch.mul(s.codes, s.scales[:, None], out=s.values)]


def _own_gemm(s):
    c = s.c

    def args(lib):
        return [s.out, c["M"], int(c["f32"]), s.x, c["K"], s.xs, s.w, c["K"], s.ws, s.bias, c["M"], c["N"], c["K"],
                *_workspace(s, lib.jllm_hip_gemm_i8_workspace(c["M"], c["N"], c["K"]))]

    _bound(s, "jllm_hip_gemm_i8", args)
    return s.out


def _own_prefix(s):
    c = s.c

    def args(lib):
        n = lib.jllm_hip_flash_attention_decode_paged_prefix_workspace(c["B"], c["heads"], c["kv"], c["hd"],
                                                                       c["prefix"], c["ctx"], c["window"])
        return [s.out, s.q, s.q.stride(0), s.kp, s.vp, s.ks, s.vs, s.n_pages, c["page"], s.prefix_table, s.prefix_len,
                c["prefix"], s.table, s.table.stride(0), s.lens, c["B"], c["heads"], c["kv"], c["hd"], c["hd"],
                c["ctx"], s.scale, int(c["int8"]), c["window"], *_workspace(s, n)]

    _bound(s, "jllm_hip_flash_attention_decode_paged_prefix", args)
    return s.out


# ---- the plain forms --------------------------------------------------------------

def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _plain_norms(s):
    c = s.c
    t = s.x.float()
    if s.post is not None:
        t = _normed(t, s.post)
    if s.gate is not None:
        g = s.gate.float()
        t = t * (g, 1 / (1 + (-g).exp()), g.tanh())[c["act"]]
    h = s.residual.float() * c["res"] + t * c["branch"]
    s.h.copy_(h)
    y = _normed(h, s.pre)
    if not c["codes"]:
        s.y.copy_(y)
        return _norms_outputs(s)
    top = y.abs().amax(-1, keepdim=True)
    s.scales.copy_(top[:, 0] / 127)
    s.codes.copy_(torch.where(top > 0, torch.round(y * (127 / top)), 0))
    return _norms_outputs(s)


def _plain_gemm(s):
    y = torch.matmul(s.x.float(), s.w.float().t()) * s.xs[:, None] * s.ws
    if s.bias is not None:
        y = y + s.bias
    return y if s.c["f32"] else y.half()


def _plain_prefix(s):
    c = s.c
    B, H, KV, hd, page, P = c["B"], c["heads"], c["kv"], c["hd"], c["page"], c["prefix"]
    G = H // KV
    q = s.q.float().view(B, KV, G, hd)
    lens = s.lens[:, None]

    def keys(slot):
        k, v = s.kp.view(-1, KV, hd)[slot].float(), s.vp.view(-1, KV, hd)[slot].float()
        if c["int8"]:
            k, v = k * s.ks.view(-1, KV)[slot][..., None], v * s.vs.view(-1, KV)[slot][..., None]
        return k, v

    # the prefix, of which a window may leave a row the last keys only
    pos = torch.arange(P, device=DEV)
    seen = (lens >= 0) & ((pos >= P + lens - c["window"]) if c["window"] else (pos >= 0))
    k, v = keys(s.prefix_table[pos // page].long() * page + pos % page)
    qp = q.permute(1, 0, 2, 3).reshape(KV, B * G, hd)
    x = torch.matmul(qp, k.permute(1, 2, 0).contiguous()).view(KV, B, G, P).permute(1, 0, 2, 3) * s.scale
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    # its own keys
    at = torch.arange(c["ctx"], device=DEV)
    live = at < lens
    if c["window"]:
        live &= at >= lens - c["window"]
    ko, vo = keys(s.table[:, at // page].clamp(min=0).long() * page + at % page)
    y = torch.matmul(q, ko.permute(0, 2, 3, 1).contiguous()) * s.scale
    y = y.masked_fill(~live[:, None, None], -math.inf)
    top = torch.maximum(x.amax(-1, keepdim=True), y.amax(-1, keepdim=True))
    top = torch.where(top.isfinite(), top, 0)
    x, y = (x - top).exp(), (y - top).exp()
    den = x.sum(-1, keepdim=True) + y.sum(-1, keepdim=True)
    num = torch.matmul(x.permute(1, 0, 2, 3).reshape(KV, B * G, P), v.transpose(0, 1).contiguous())
    num = num.view(KV, B, G, hd).permute(1, 0, 2, 3) + torch.matmul(y, vo.transpose(1, 2).contiguous())
    return torch.where(den > 0, num / den, 0).reshape(B, H * hd).half()


# ---- the definitions in 64 bits ---------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"norms": _exact_norms, "gemm": _exact_gemm, "prefix": _exact_prefix}[s.kind](s, case)


def _exact_norms(s, c):
    def rms(x, w):
        return x / (x.pow(2).sum(1, keepdim=True) / c["hidden"] + EPS).sqrt() * w.to(torch.float64)

    t = s.x.to(torch.float64)
    t = rms(t, s.post) if c["post"] else t
    if c["gate"]:
        g = s.gate.to(torch.float64)
        t = t * [lambda: g, lambda: torch.sigmoid(g), lambda: torch.tanh(g)][c["act"]]()
    h = torch.add(s.residual.to(torch.float64) * c["res"], t, alpha=c["branch"])
    y = rms(h, s.pre)
    if c["codes"]:
        step = y.abs().amax(1, keepdim=True) / 127
        y = torch.round(y / step) * step
    return [h, y]


def _exact_gemm(s, c):
    # whole numbers below 2^53: the sums are exact in 64 bits
    w = s.w.to(torch.float64).t().contiguous()
    y = s.x.to(torch.float64) @ w
    y = torch.outer(s.xs.to(torch.float64), s.ws.to(torch.float64)) * y
    return y if s.bias is None else y + s.bias.to(torch.float64)


def _exact_prefix(s, c):
    KV, hd, page, P, w = c["kv"], c["hd"], c["page"], c["prefix"], c["window"]

    def rows(pool, scales, ids, n):
        x = pool[ids.long()].reshape(-1, KV, hd)[:n].to(torch.float64)
        x = x if scales is None else x * scales[ids.long()].reshape(-1, KV, 1)[:n].to(torch.float64)
        return x.transpose(0, 1).contiguous()

    pk, pv = rows(s.kp, s.ks, s.prefix_table, P), rows(s.vp, s.vs, s.prefix_table, P)

    def row(b, n):
        if n < 0:
            return torch.zeros((c["heads"] * hd,), dtype=torch.float64, device=DEV)
        ids = s.table[b, :_pages(c, n)]
        k = torch.cat([pk, rows(s.kp, s.ks, ids, n)], 1)
        v = torch.cat([pv, rows(s.vp, s.vs, ids, n)], 1)
        lo = max(0, P + n - w) if w else 0
        q = s.q[b].to(torch.float64).view(KV, -1, hd)
        out = []
        for h in range(KV):
            p = torch.softmax((q[h] @ k[h, lo:].t().contiguous()) / math.sqrt(hd), -1)
            out.append(p @ v[h, lo:])
        return torch.cat(out).flatten()

    return torch.stack([row(b, n) for b, n in enumerate(s.lens.tolist())])


# ---- what a pass cannot do without ------------------------------------------------

def work(c):
    if c["kind"] == "norms":
        n, wide = c["rows"] * c["hidden"], 4 if c["wide"] else 2
        gate = 2 * (n if c["gate"] == "rows" else c["hidden"]) if c["gate"] else 0
        vectors = c["hidden"] * (8 if c["post"] else 4)
        return {"bytes": n * (2 + 2 * wide + (1 if c["codes"] else 2)) + gate + vectors +
                (4 * c["rows"] if c["codes"] else 0), "flops": 8 * n}
    if c["kind"] == "gemm":
        N, M, K = c["N"], c["M"], c["K"]
        return {"bytes": (N + M) * K + 4 * (N + M) + (4 * M if c["bias"] else 0) + N * M * (4 if c["f32"] else 2),
                "flops": 2 * N * M * K}
    B, H, KV, hd, P, w = c["B"], c["heads"], c["kv"], c["hd"], c["prefix"], c["window"]
    lens = [n for n in _own_lengths(c) if n >= 0]
    behind = sum(min(n, w) if w else n for n in lens)
    before = [max(0, min(P, w - n)) if w else P for n in lens]
    size = 2 * KV * (hd + 4 if c["int8"] else 2 * hd)
    return {"bytes": (max(before, default=0) + behind) * size + 4 * (_pages(c, P) + sum(_pages(c, n) for n in lens)) +
            B * (4 * H * hd + 4), "flops": 4 * H * hd * (sum(before) + behind)}
