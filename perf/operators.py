"""Performance cases of the batched serving operators: the attention front that stores
into a paged KV cache, decode attention over the pages, and the processing of a
batch's logits, each through its public entry point (the C ABI of
include/jllm_hip.h) or, where `own` is false, in its plain form.

Head layouts are those of the repository's decoder configuration (32 / 8 heads x 128,
vocabulary 151936) and of its tests; `draw` spreads over the ranges around them.

A case's "kind":
  front    q / k norm, rotation and KV store of N tokens (qk_norm_rope_store_kv_paged)
  attn     one query row of each of B sequences over its pages (flash_attention_decode_paged)
  logits   penalties, biases and masks of B rows, with the greedy token (logits_process)
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
EPS, THETA = 1e-6, 1e6
VOCAB = 151936


def listed():
    return [
        # one user's decode step: a single token, where latency is all there is
        _front("front_one", N=1),
        # decode step of a full batch, four rows of padding behind it, q / k / v in one fused buffer
        _front("front_batch", N=64, fused=True, pad=4),
        # a prompt chunk into an INT8 cache
        _front("front_prompt", N=2048, int8=True, fused=True),
        # ragged prompts of a small-headed model without q / k norms, interleaved pairs
        _front("front_pairs", N=7777, heads=8, kv=2, hd=64, neox=False, norm=False),
        # decode attention in the chat regime, one user
        _attn("attn_one", B=1, ctx=700, int8=True),
        # a full batch of chats of different lengths, two padded rows among them
        _attn("attn_batch", B=48, ctx=4096, int8=True, ragged=True),
        # one long document
        _attn("attn_long", B=1, ctx=131072, page=64),
        # a batch of long documents in an fp16 cache: the largest read
        _attn("attn_large", B=24, ctx=16384, page=32, ragged=True),
        # sliding-window layers, one KV head for twelve query heads
        _attn("attn_window", B=17, ctx=5000, heads=12, kv=1, hd=96, window=1024, ragged=True),
        # one user's logits: a chat's history, no grammar
        _logits("logits_one", B=1, hist=700),
        # a batch of requests with histories, biases and grammar masks
        _logits("logits_batch", B=64, hist=4096, bias=100, mask=True),
        # a large batch over an odd vocabulary, rows not aligned
        _logits("logits_odd", B=251, V=32003, hist=300, bias=7, mask=True),
    ]


def _front(name, N, heads=32, kv=8, hd=128, int8=False, neox=True, norm=True, fused=False, pad=0):
    c = {"kind": "front", "N": N, "heads": heads, "kv": kv, "hd": hd, "int8": int8, "neox": neox, "norm": norm,
         "fused": fused, "pad": pad}
    return dict(c, name=name) if name else c


def _attn(name, B, ctx, heads=32, kv=8, hd=128, page=16, int8=False, window=0, ragged=False):
    c = {"kind": "attn", "B": B, "ctx": ctx, "heads": heads, "kv": kv, "hd": hd, "page": page, "int8": int8,
         "window": window, "ragged": ragged}
    return dict(c, name=name) if name else c


def _logits(name, B, V=VOCAB, hist=0, bias=0, mask=False):
    c = {"kind": "logits", "B": B, "V": V, "hist": hist, "bias": bias, "mask": mask}
    return dict(c, name=name) if name else c


def _logint(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["front", "attn", "attn", "logits"])
    heads, kv, hd = rng.choice([(32, 8, 128), (32, 8, 128), (16, 4, 128), (16, 2, 128), (8, 2, 64), (8, 8, 64),
                                (12, 1, 96), (4, 1, 32)])
    int8 = rng.random() < 0.5
    if kind == "front":
        N = _logint(rng, 1, 8000)
        return _front("", N, heads, kv, hd, int8, rng.random() < 0.7, rng.random() < 0.7, rng.random() < 0.5,
                      rng.choice([0, 0, rng.randint(0, 9)]))
    if kind == "attn":
        B = _logint(rng, 1, 64)
        ctx = _logint(rng, 1, min(131072, 390000 // B))
        return _attn("", B, ctx, heads, kv, hd, rng.choice([16, 16, 32, 64, 256]), int8,
                     rng.choice([0, 0, _logint(rng, 1, 4096)]), rng.random() < 0.7)
    V = rng.choice([VOCAB, rng.randint(1000, VOCAB), rng.randint(1000, VOCAB)])
    return _logits("", _logint(rng, 1, min(256, 9700000 // V)), V, rng.choice([0, _logint(rng, 1, 8192)]),
                   rng.choice([0, rng.randint(1, 300)]), rng.random() < 0.5)


# ---- inputs -----------------------------------------------------------------------

class State:
    pass


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def _lengths(n, most, ragged):
    """Lengths of a batch's rows: the longest is `most`, half of the others are anywhere
    below it, the other half short (spread over its logarithm), every 23rd row is
    padding (length 0)."""
    if not ragged:
        return [most] * n
    r = random.Random("%d %d" % (n, most))
    return [most if i == 0 else 0 if i % 23 == 22 else r.randint(1, most) if i % 2 else _logint(r, 1, most)
            for i in range(n)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    return {"front": _prepare_front, "attn": _prepare_attn, "logits": _prepare_logits}[case["kind"]](case, seed)


def _prepare_front(c, seed):
    g, s = _gen(seed), State()
    s.c, s.kind = c, "front"
    N, H, KV, hd = c["N"], c["heads"], c["kv"], c["hd"]
    rows = N + c["pad"]
    qkv = (_randn(g, rows, (H + 2 * KV) * hd) * 1.5).half()
    s.q, s.k, s.v = qkv.split([H * hd, KV * hd, KV * hd], dim=1)
    if not c["fused"]:
        s.q, s.k, s.v = s.q.contiguous(), s.k.contiguous(), s.v.contiguous()
    s.qw = s.kw = None
    if c["norm"]:
        s.qw, s.kw = (1 + 0.2 * _randn(g, hd), 1 + 0.2 * _randn(g, hd))
    # prompts put consecutive positions, decode steps one far position of each sequence
    s.pos = (torch.arange(rows, device=DEV) if N > 256 else
             torch.randint(0, 131072, (rows,), device=DEV, generator=g)).int()
    s.n_slots = 16 * ((rows + rows // 4) // 16 + 1)
    s.slots = torch.randperm(s.n_slots, device=DEV, generator=g)[:rows].int()
    s.slots[N:] = -1
    s.q_out = torch.zeros((rows, H * hd), dtype=torch.float16, device=DEV)
    kind = torch.int8 if c["int8"] else torch.float16
    s.kp, s.vp = (torch.zeros((s.n_slots, KV, hd), dtype=kind, device=DEV) for _ in range(2))
    s.ks = s.vs = None
    if c["int8"]:
        s.ks, s.vs = (torch.zeros((s.n_slots, KV), device=DEV) for _ in range(2))
        s.kf, s.vf = (torch.zeros((s.n_slots, KV, hd), dtype=torch.float16, device=DEV) for _ in range(2))
    return s


def _pages_of(c):
    return [(n + c["page"] - 1) // c["page"] for n in _lengths(c["B"], c["ctx"], c["ragged"])]


def _prepare_attn(c, seed):
    g, s = _gen(seed), State()
    s.c, s.kind = c, "attn"
    B, H, KV, hd, page = c["B"], c["heads"], c["kv"], c["hd"], c["page"]
    lens, used = _lengths(B, c["ctx"], c["ragged"]), _pages_of(c)
    s.n_pages = sum(used) + 3
    s.lens = _ints(lens)
    s.width = max(used)
    # every sequence's pages lie anywhere in the pool; entries behind its last page are -1
    ids = torch.randperm(s.n_pages, device=DEV, generator=g).int()[:sum(used)]
    at = torch.arange(s.width, device=DEV)[None] < _ints(used)[:, None]
    s.table = torch.full((B, s.width), -1, dtype=torch.int32, device=DEV)
    s.table[at] = ids
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


def _prepare_logits(c, seed):
    g, s = _gen(seed), State()
    s.c, s.kind = c, "logits"
    B, V = c["B"], c["V"]
    s.x = _randn(g, B, V) * 3
    s.out = torch.zeros((B, V), device=DEV)
    s.tok = torch.zeros((B,), dtype=torch.int32, device=DEV)
    s.hist = s.n_prompt = s.n_hist = s.rep = s.freq = s.pres = None
    if c["hist"]:
        n = _lengths(B, c["hist"], True)
        s.n_hist, s.n_prompt = _ints(n), _ints([x // 2 for x in n])
        # a text repeats itself: ids crowd at the low end of the vocabulary
        u = torch.rand((B, c["hist"]), device=DEV, generator=g)
        s.hist = (u.pow(3) * V).int().clamp_(0, V - 1)
        s.rep = 1 + torch.rand((B,), device=DEV, generator=g) * 0.3
        s.freq = torch.rand((B,), device=DEV, generator=g) * 0.5
        s.pres = torch.rand((B,), device=DEV, generator=g) * 0.5
    s.bias_ids = s.bias = s.n_bias = None
    if c["bias"]:
        s.bias_ids = torch.randint(0, V, (B, c["bias"]), dtype=torch.int32, device=DEV, generator=g)
        s.bias = _randn(g, B, c["bias"]) * 5
        s.n_bias = _ints(_lengths(B, c["bias"], True))
    s.mask = None
    if c["mask"]:
        # every third row's grammar allows a few tokens, the others most of the vocabulary
        words = (V + 31) // 32
        s.mask = torch.randint(-2 ** 31, 2 ** 31, (B, words), dtype=torch.int32, device=DEV, generator=g)
        s.mask |= torch.randint(-2 ** 31, 2 ** 31, (B, words), dtype=torch.int32, device=DEV, generator=g)
        few = torch.rand((B, words), device=DEV, generator=g) < 0.005
        strict = torch.arange(B, device=DEV)[:, None] % 3 == 1
        s.mask = torch.where(strict & ~few, torch.zeros_like(s.mask), s.mask)
    return s


# ---- one pass ---------------------------------------------------------------------

def run(s):
    if own:
        return {"front": _own_front, "attn": _own_attn, "logits": _own_logits}[s.kind](s)
    return {"front": _plain_front, "attn": _plain_attn, "logits": _plain_logits}[s.kind](s)


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


def _own_front(s):
    c = s.c

    def args(lib):
        return [s.q_out, s.q_out.stride(0), s.q, s.q.stride(0), s.k, s.k.stride(0), s.v, s.v.stride(0),
                s.qw, s.kw, 1, EPS, s.kp, s.vp, s.ks, s.vs, s.n_slots, s.pos, s.slots,
                c["heads"], c["kv"], c["hd"], c["hd"], s.q.shape[0], THETA, int(c["neox"]), int(c["int8"])]

    _bound(s, "jllm_hip_qk_norm_rope_store_kv_paged", args)
    return _front_outputs(s, s.q_out)


def _front_outputs(s, q):
    if not s.c["int8"]:
        return [q, s.kp, s.vp]
    # codes as the values they stand for
    return [q, torch.mul(s.kp, s.ks[..., None], out=s.kf), torch.mul(s.vp, s.vs[..., None], out=s.vf)]


def _own_attn(s):
    c = s.c

    def args(lib):
        n = lib.jllm_hip_flash_attention_decode_paged_workspace(c["B"], c["heads"], c["kv"], c["hd"], c["ctx"],
                                                                c["window"])
        s.ws = torch.empty((max(n, 16),), dtype=torch.uint8, device=DEV)
        return [s.out, s.q, s.q.stride(0), s.kp, s.vp, s.ks, s.vs, s.n_pages, c["page"], s.table, s.table.stride(0),
                s.lens, c["B"], c["heads"], c["kv"], c["hd"], c["hd"], c["ctx"], s.scale, int(c["int8"]),
                c["window"], s.ws, s.ws.numel()]

    _bound(s, "jllm_hip_flash_attention_decode_paged", args)
    return s.out


def _own_logits(s):
    c = s.c

    def args(lib):
        s.ws = torch.empty((max(lib.jllm_hip_logits_process_workspace(c["B"], c["V"]), 16),), dtype=torch.uint8,
                           device=DEV)
        return [s.out, c["V"], s.x, c["V"], c["B"], c["V"], s.hist, c["hist"], s.n_prompt, s.n_hist, s.rep, s.freq,
                s.pres, s.bias_ids, s.bias, c["bias"], s.n_bias, s.mask, (c["V"] + 31) // 32, s.tok, s.ws,
                s.ws.numel()]

    _bound(s, "jllm_hip_logits_process", args)
    return [s.out, s.tok]


# ---- the plain forms --------------------------------------------------------------

def _normed(x, w):
    if w is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _rotated(x, cos, sin, neox):
    h = x.shape[-1] // 2
    a, b = (x[..., :h], x[..., h:]) if neox else (x[..., 0::2], x[..., 1::2])
    u, w = a * cos - b * sin, a * sin + b * cos
    return torch.cat([u, w], -1) if neox else torch.stack([u, w], -1).flatten(-2)


def _plain_front(s):
    c = s.c
    rows, H, KV, hd = s.q.shape[0], c["heads"], c["kv"], c["hd"]
    # far positions: the angle keeps 64 bits up to its sine and cosine
    inv = THETA ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    ang = s.pos.double()[:, None, None] * inv
    cos, sin = ang.cos().float(), ang.sin().float()
    q = _rotated(_normed(s.q.float().reshape(rows, H, hd), s.qw), cos, sin, c["neox"])
    k = _rotated(_normed(s.k.float().reshape(rows, KV, hd), s.kw), cos, sin, c["neox"])
    live = (s.slots >= 0) & (s.slots < s.n_slots)
    at = s.slots[live].long()
    q = torch.where(live[:, None], q.reshape(rows, -1).half(), s.q_out)
    k, v = k[live], s.v.float().reshape(rows, KV, hd)[live]
    if not c["int8"]:
        s.kp[at], s.vp[at] = k.half(), v.half()
        return _front_outputs(s, q)
    km, vm = k.abs().amax(-1, keepdim=True), v.abs().amax(-1, keepdim=True)
    s.ks[at], s.vs[at] = km[..., 0] / 127, vm[..., 0] / 127
    s.kp[at] = torch.where(km > 0, torch.round(k * (127 / km)), 0).to(torch.int8)
    s.vp[at] = torch.where(vm > 0, torch.round(v * (127 / vm)), 0).to(torch.int8)
    return _front_outputs(s, q)


def _plain_attn(s):
    c = s.c
    B, H, KV, hd, page = c["B"], c["heads"], c["kv"], c["hd"], c["page"]
    pos = torch.arange(c["ctx"], device=DEV)
    lens = s.lens[:, None]
    live = pos < lens
    if c["window"]:
        live &= pos >= lens - c["window"]
    slot = s.table[:, pos // page].clamp(min=0).long() * page + pos % page
    k, v = s.kp.view(-1, KV, hd)[slot].float(), s.vp.view(-1, KV, hd)[slot].float()
    if c["int8"]:
        k, v = k * s.ks.view(-1, KV)[slot][..., None], v * s.vs.view(-1, KV)[slot][..., None]
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    x = torch.matmul(s.q.float().view(B, KV, H // KV, hd), k) * s.scale
    live = live[:, None, None, :]
    top = x.masked_fill(~live, -math.inf).amax(-1, keepdim=True)
    p = torch.where(live, (x - top).exp(), 0)
    den = p.sum(-1, keepdim=True)
    out = torch.where(den > 0, torch.matmul(p, v) / den, 0)
    return out.reshape(B, H * hd).half()


def _plain_logits(s):
    c = s.c
    B, V = c["B"], c["V"]
    y = s.x
    if s.hist is not None:
        place = torch.arange(c["hist"], device=DEV)[None]
        ids = s.hist.long()
        counted = (place < s.n_hist[:, None]) & (place >= s.n_prompt[:, None])
        n = torch.zeros((B, V), device=DEV).scatter_add_(1, ids, counted.float())
        seen = torch.zeros((B, V), device=DEV).scatter_add_(1, ids, (place < s.n_hist[:, None]).float()) > 0
        r = s.rep[:, None]
        y = torch.where(seen, torch.where(y > 0, y / r, y * r), y)
        y = y - s.freq[:, None] * n
        y = torch.where(n > 0, y - s.pres[:, None], y)
    if s.bias_ids is not None:
        # of a token that a row lists twice the last bias counts
        place = torch.arange(c["bias"], device=DEV)[None]
        nth = torch.where(place < s.n_bias[:, None], place + 1, 0)
        last = torch.zeros((B, V), dtype=torch.long, device=DEV).scatter_reduce_(1, s.bias_ids.long(), nth, "amax")
        y = torch.where(last > 0, y + s.bias.gather(1, (last - 1).clamp(min=0)), y)
    if s.mask is not None:
        v = torch.arange(V, device=DEV)
        y = torch.where((s.mask[:, v >> 5] >> (v & 31).int()) & 1 == 1, y, -math.inf)
    fine = torch.where(y.isfinite(), y, -math.inf)
    top = fine.amax(-1, keepdim=True)
    at = torch.where((fine == top) & fine.isfinite(), torch.arange(V, device=DEV), V).amin(-1)
    return [y, torch.where(at < V, at, -1).int()]


# ---- the definitions in 64 bits ---------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"front": _exact_front, "attn": _exact_attn, "logits": _exact_logits}[s.kind](s, case)


def _exact_front(s, c):
    hd, half = c["hd"], c["hd"] // 2
    inv = torch.tensor([THETA ** (-2.0 * i / hd) for i in range(half)], dtype=torch.float64, device=DEV)
    turn = torch.exp(1j * (s.pos.to(torch.float64)[:, None] * inv).to(torch.complex128))[:, None]

    def heads(x, n):
        return x.to(torch.float64).reshape(len(x), n, hd)

    def turned(x, w):
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.to(torch.float64)
        z = torch.complex(x[..., :half], x[..., half:]) if c["neox"] else torch.view_as_complex(
            x.unflatten(-1, (half, 2)).contiguous())
        z = z * turn
        return torch.cat([z.real, z.imag], -1) if c["neox"] else torch.view_as_real(z).flatten(-2)

    n = c["N"]
    q = torch.zeros(s.q_out.shape, dtype=torch.float64, device=DEV)
    q[:n] = turned(heads(s.q, c["heads"]), s.qw).flatten(1)[:n]
    out = [q]
    for x in (turned(heads(s.k, c["kv"]), s.kw), heads(s.v, c["kv"])):
        if c["int8"]:
            step = x.abs().amax(-1, keepdim=True) / 127
            x = torch.round(x / step) * step
        pool = torch.zeros(s.kp.shape, dtype=torch.float64, device=DEV)
        pool.index_copy_(0, s.slots[:n].long(), x[:n])
        out.append(pool)
    return out


def _exact_attn(s, c):
    H, KV, hd, page = c["heads"], c["kv"], c["hd"], c["page"]

    def rows(pool, scales, ids, lo, n):
        x = pool[ids].reshape(-1, KV, hd)[lo:n].to(torch.float64)
        return (x if scales is None else x * scales[ids].reshape(-1, KV, 1)[lo:n].to(torch.float64)).transpose(0, 1)

    def head(q, k, v):
        return torch.softmax((q @ k.T.contiguous()) / math.sqrt(hd), -1) @ v.contiguous()

    def row(b, n):
        if n == 0:
            return torch.zeros((H * hd,), dtype=torch.float64, device=DEV)
        lo = max(0, n - c["window"]) if c["window"] else 0
        ids = s.table[b, :(n + page - 1) // page].long()
        k, v = rows(s.kp, s.ks, ids, lo, n), rows(s.vp, s.vs, ids, lo, n)
        q = s.q[b].to(torch.float64).view(KV, H // KV, hd)
        return torch.cat([head(*x) for x in zip(q, k, v)]).flatten()

    return torch.stack([row(b, n) for b, n in enumerate(s.lens.tolist())])


def _exact_logits(s, c):
    V = c["V"]

    def row(b):
        y = s.x[b].to(torch.float64)
        if s.hist is not None:
            n, p = int(s.n_hist[b]), int(s.n_prompt[b])
            n_out = torch.bincount(s.hist[b, p:n].long(), minlength=V)
            old = (torch.bincount(s.hist[b, :p].long(), minlength=V) + n_out) > 0
            r = s.rep[b].to(torch.float64)
            y[old] = torch.where(y[old] > 0, y[old] / r, y[old] * r)
            y -= s.freq[b].to(torch.float64) * n_out + s.pres[b].to(torch.float64) * (n_out > 0)
        if s.bias_ids is not None:
            m = int(s.n_bias[b])
            last = dict(zip(s.bias_ids[b, :m].tolist(), s.bias[b, :m].tolist()))
            y[list(last)] += torch.tensor(list(last.values()), dtype=torch.float64, device=DEV)
        if s.mask is not None:
            bits = (s.mask[b].unsqueeze(1) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
            y[bits.flatten()[:V] == 0] = -math.inf
        return y

    y = torch.stack([row(b) for b in range(c["B"])])
    best = y.argmax(-1)
    return [y, torch.where(y.amax(-1).isfinite(), best, -1).int()]


# ---- what a pass cannot do without ------------------------------------------------

def work(c):
    if c["kind"] == "front":
        N, H, KV, hd = c["N"], c["heads"], c["kv"], c["hd"]
        row = hd + 4 if c["int8"] else 2 * hd
        return {"bytes": N * (2 * (H + 2 * KV) * hd + 2 * H * hd + 2 * KV * row + 8), "flops": N * (H + KV) * hd * 8}
    if c["kind"] == "attn":
        H, KV, hd = c["heads"], c["kv"], c["hd"]
        row = hd + 4 if c["int8"] else 2 * hd
        keys = sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c["B"], c["ctx"], c["ragged"]))
        return {"bytes": keys * 2 * KV * row + 4 * sum(_pages_of(c)) + c["B"] * (4 * H * hd + 4),
                "flops": 4 * keys * H * hd}
    B, V = c["B"], c["V"]
    lists = 4 * sum(_lengths(B, c["hist"], True)) if c["hist"] else 0
    bias = 8 * sum(_lengths(B, c["bias"], True)) if c["bias"] else 0
    return {"bytes": 8 * B * V + lists + bias + (B * 4 * ((V + 31) // 32) if c["mask"] else 0), "flops": 4 * B * V}
