"""The serving operators over a paged K/V cache, and beam search on it, as performance cases.

The kinds:

  plan     pages, slots and positions of a step's new tokens from the requests' lengths
  append   the new tokens' K and V rows into their slots
  attn     attention of a chunk of new tokens (one or many a request) over the cache
  beam     the selection of the next beams over beams and vocabulary
  reorder  the beams' block tables after a selection, with the copies of their open pages

A case is a dict of plain values; prepare() makes its inputs on the GPU from the seed
alone, run() is one pass: through the C ABI of include/cdml.h where `own` is set, in
elementary torch operations otherwise.  exact() gives the same results in float64.
"""
from __future__ import annotations

import ctypes
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")


def listed():
    return [
        # long-context serving: one new token for each of 64 requests of 8192 tokens
        {"name": "attn_decode_long", "kind": "attn", "batch": 64, "new": 1, "kv": 8192, "full": True, "heads": 16,
         "kv_heads": 16, "hd": 128, "page": 64, "type": "f32"},
        # a few requests that are being generated, 16-bit cache: the call's latency counts
        {"name": "attn_decode_few", "kind": "attn", "batch": 8, "new": 1, "kv": 2048, "full": True, "heads": 16,
         "kv_heads": 16, "hd": 64, "page": 16, "type": "bf16"},
        # whole prompts of 4096 tokens
        {"name": "attn_prompts", "kind": "attn", "batch": 4, "new": 4096, "kv": 4096, "full": True, "heads": 16,
         "kv_heads": 16, "hd": 64, "page": 16, "type": "f32"},
        # chunked prefill of ragged requests, some idle, grouped heads, 16-bit cache
        {"name": "attn_chunks", "kind": "attn", "batch": 24, "new": 311, "kv": 5003, "full": False, "heads": 32,
         "kv_heads": 8, "hd": 128, "page": 32, "type": "bf16"},
        # a decode step of 64 requests in a pool of half a million tokens
        {"name": "plan_decode", "kind": "plan", "batch": 64, "new": 1, "kv": 8192, "max": 16384, "page": 16,
         "pages": 40000},
        # many prompts of ragged lengths at once
        {"name": "plan_prompts", "kind": "plan", "batch": 250, "new": 1021, "kv": 0, "max": 2048, "page": 16,
         "pages": 40000},
        # one row a request
        {"name": "append_decode", "kind": "append", "rows": 64, "dim": 2048, "page": 64, "pages": 256, "type": "f32"},
        # four prompts of 4096 tokens into a 16-bit cache
        {"name": "append_prompts", "kind": "append", "rows": 16384, "dim": 1024, "page": 16, "pages": 1500,
         "type": "bf16"},
        # the small text model's beams
        {"name": "beam_small", "kind": "beam", "batch": 4, "beams": 4, "vocab": 200, "alpha": 0.0},
        # many wide beams over a large vocabulary, some of them finished
        {"name": "beam_large", "kind": "beam", "batch": 64, "beams": 8, "vocab": 50021, "alpha": 0.6},
        # the small text model's tables after a selection
        {"name": "reorder_small", "kind": "reorder", "batch": 4, "beams": 4, "kv": 60, "dim": 64, "page": 16,
         "layers": 2, "type": "f32"},
        # many wide beams on long prompts
        {"name": "reorder_large", "kind": "reorder", "batch": 64, "beams": 8, "kv": 2037, "dim": 512, "page": 16,
         "layers": 2, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# No drawn case costs more than the largest listed one of its sort.
_MOST = {"flops": 1.2e11, "bytes": 8.7e9, "scores": 1.1e9}


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        scores = case["batch"] * case["heads"] * case["new"] * case["kv"] if case["kind"] == "attn" else 0
        if w["flops"] <= _MOST["flops"] and w["bytes"] <= _MOST["bytes"] and scores <= _MOST["scores"]:
            return case


def _draw(rng):
    kind = rng.choice(("plan", "append", "attn", "attn", "attn", "attn", "beam", "reorder"))
    page, dtype = rng.choice((8, 16, 16, 32, 64, 128)), rng.choice(("f32", "bf16", "bf16", "f16"))
    if kind == "attn":
        heads, kv_heads = rng.choice(((16, 16), (8, 8), (5, 5), (1, 1), (32, 8), (16, 2), (12, 4), (7, 1)))
        kv = _log(rng, 1, 8192)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, kv)
        return {"kind": kind, "batch": _log(rng, 1, 64), "new": new, "kv": kv, "full": rng.random() < 0.3,
                "heads": heads, "kv_heads": kv_heads, "hd": rng.choice((8, 16, 32, 40, 64, 64, 96, 128, 128)),
                "page": page, "type": dtype}
    if kind == "plan":
        batch, most = _log(rng, 1, 512), _log(rng, 16, 8192)
        kv = rng.choice((0, most // 2))
        return {"kind": kind, "batch": batch, "new": 1 if rng.random() < 0.5 else max(1, (most - kv) // 3), "kv": kv,
                "max": most, "page": page, "pages": batch * -(-most // page) + 8}
    if kind == "append":
        rows = _log(rng, 1, 16384)
        return {"kind": kind, "rows": rows, "dim": rng.choice((8, 64, 96, 200, 256, 512, 1000, 1024, 2048)),
                "page": page, "pages": -(-rows * 5 // (4 * page)) + 1, "type": dtype}
    if kind == "beam":
        return {"kind": kind, "batch": _log(rng, 1, 64), "beams": rng.randint(1, 12), "vocab": _log(rng, 20, 50000),
                "alpha": rng.choice((0.0, 0.6, 1.0))}
    return {"kind": kind, "batch": _log(rng, 1, 64), "beams": rng.randint(2, 12), "kv": _log(rng, 1, 4096),
            "dim": rng.choice((64, 200, 512)), "page": page, "layers": rng.randint(1, 3), "type": dtype}


def work(case):
    """Bytes (each input read once, each output written once, pages' visible tokens only) and flops
    (two per multiply-add, visible query-key pairs only; five per logit of a selection) of one pass."""
    c, k = case, case["kind"]
    if k == "attn":
        lens, news = _lengths(c)
        size, seen = _bytes_of(c["type"]), sum(n * m - n * (n - 1) // 2 for m, n in zip(lens, news))
        cache = sum(m for m, n in zip(lens, news) if n) * 2 * c["kv_heads"] * c["hd"] * size
        return {"bytes": cache + 8 * sum(news) * c["heads"] * c["hd"], "flops": 4 * c["hd"] * c["heads"] * seen}
    if k == "plan":
        lens, news = _lengths(c)
        return {"bytes": 4 * (c["pages"] + 4 * c["batch"] + 2 * sum(news) + 2 * sum(news) // c["page"]), "flops": 0}
    if k == "append":
        return {"bytes": c["rows"] * (c["dim"] * (8 + 2 * _bytes_of(c["type"])) + 4), "flops": 0}
    if k == "beam":
        rows = c["batch"] * c["beams"]
        return {"bytes": 4 * rows * c["vocab"] + 22 * rows, "flops": 5 * rows * c["vocab"]}
    rows, blocks = c["batch"] * c["beams"], -(-c["kv"] // c["page"])
    # every second row copies, of half a page
    copied = rows // 2 * (c["page"] // 2) * c["dim"] * _bytes_of(c["type"]) * 4 * c["layers"]
    return {"bytes": 8 * rows * blocks + 28 * rows + copied, "flops": 0}


def _bytes_of(name):
    return 4 if name == "f32" else 2


def _lengths(c):
    """Tokens of each request with the new ones, and how many are new: all the same, or spread from none to the
    largest, every fifth request with one new token and every seventh idle (plan: tokens before the step)."""
    if c["kind"] == "plan":
        kv = [(c["kv"] * (7 * b + 3)) % (c["kv"] + 1) if c["kv"] else 0 for b in range(c["batch"])]
        return kv, [1 + (37 * b + 11) % c["new"] for b in range(c["batch"])]
    if c["full"]:
        return [c["kv"]] * c["batch"], [min(c["new"], c["kv"])] * c["batch"]
    lens, news = [], []
    for b in range(c["batch"]):
        n = 0 if b % 7 == 6 else 1 if b % 5 == 4 else c["new"] - (29 * b) % max(1, c["new"] // 2)
        m = c["kv"] - (101 * b) % max(1, c["kv"] * 3 // 4)
        lens.append(max(m, 1))
        news.append(min(n, max(m, 1)))
    return lens, news


# ---- inputs ---------------------------------------------------------------

class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device=DEV, generator=self.g) * std).to(dtype)

    def perm(self, n):
        return torch.randperm(n, device=DEV, generator=self.g).to(torch.int32)

    def below(self, n, *shape):
        return torch.randint(0, n, shape, device=DEV, generator=self.g)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _tables(state, n_pages, blocks, rows):
    """The views of a state's flat buffer: page references, block table and lengths."""
    refs, rest = state[:n_pages], state[n_pages:]
    return refs, rest[:rows * blocks].view(rows, blocks), rest[rows * blocks:]


def prepare(case, seed):
    c, k, r = case, case["kind"], _Rand(seed)
    s = {"case": c}
    if k == "plan":
        lens, news = _lengths(c)
        blocks = -(-c["max"] // c["page"])
        kv, new = _ints(lens), _ints(news)
        have = (kv + c["page"] - 1) // c["page"]
        start = torch.cumsum(have, 0, dtype=torch.int32) - have
        order, at = r.perm(c["pages"]), torch.arange(blocks, device=DEV)[None]
        used = at < have[:, None]
        pages = order[(start[:, None] + at).clamp(max=c["pages"] - 1)]
        table = torch.where(used, pages, torch.full_like(pages, -1))
        # a quarter of the other pages belongs to requests that this step leaves out
        refs = (r.below(4, c["pages"]) == 0).to(torch.int32)
        refs[table[used].long()] = 1
        s.update(new=new, rows=sum(news) + 5, blocks=blocks, first=torch.cat([refs, table.reshape(-1), kv]))
        s["state"] = s["first"].clone()
        s["cu"], s["slots"], s["positions"] = (torch.zeros(n, dtype=torch.int32, device=DEV)
                                               for n in (c["batch"] + 1, s["rows"], s["rows"]))
        s["status"] = torch.zeros(3, dtype=torch.int32, device=DEV)
        return s
    if k == "append":
        n = c["pages"] * c["page"]
        s["k"], s["v"] = r.normal(c["rows"], c["dim"]), r.normal(c["rows"], c["dim"])
        # padding rows at the end of a step have no slot
        s["slots"] = torch.where(torch.arange(c["rows"], device=DEV) % 64 == 63, -1, r.perm(n)[:c["rows"]])
        s["slots"] = s["slots"].to(torch.int32)
        # a spare row behind each cache takes the plain form's padding
        s["kc"], s["vc"] = (torch.zeros(n + 1, c["dim"], device=DEV, dtype=TYPES[c["type"]]) for _ in range(2))
        return s
    if k == "attn":
        lens, news = _lengths(c)
        P, D = c["page"], c["kv_heads"] * c["hd"]
        blocks = -(-max(lens) // P)
        n_pages = c["batch"] * blocks
        # ragged steps end in a few padding rows
        s.update(lens=lens, news=news, blocks=blocks, pages=n_pages, rows=sum(news) + (0 if c["full"] else 3))
        s["q"] = r.normal(s["rows"], c["heads"] * c["hd"])
        s["o"] = torch.zeros_like(s["q"])
        s["kc"], s["vc"] = (r.normal(n_pages * P, D, dtype=TYPES[c["type"]]) for _ in range(2))
        s["table"] = r.perm(n_pages).view(c["batch"], blocks)
        s["kv_len"] = _ints(lens)
        s["cu"] = _ints([0] + list(np.cumsum(news)))
        s["bad"] = torch.zeros(1, dtype=torch.int32, device=DEV)
        return s
    if k == "beam":
        R = c["batch"] * c["beams"]
        # a peaked distribution, as a trained model's logits have
        s["x"] = r.normal(R, c["vocab"], std=2.0)
        likely = (r.below(c["vocab"], R, 1) + torch.arange(8, device=DEV) * (c["vocab"] // 8)) % c["vocab"]
        s["x"].scatter_(1, likely, r.normal(R, 8, std=4.0).abs() + 2)
        s["score"] = r.normal(R, std=3.0).abs().neg() - 5
        s["len"] = (r.below(20, R) + 3).to(torch.int32)
        s["done"] = (r.below(8, R) == 0).to(torch.uint8)
        s["out"] = {"score": torch.zeros(R, device=DEV), "len": torch.zeros_like(s["len"]),
                    "done": torch.zeros_like(s["done"]), "parent": torch.zeros_like(s["len"]),
                    "token": torch.zeros_like(s["len"])}
        return s
    B, K, P = c["batch"], c["beams"], c["page"]
    R, blocks = B * K, -(-c["kv"] // P) + 1
    # the beams of a prompt share the pages of its first seven eighths and own the rest
    lens = np.array([max(0, c["kv"] - 13 * b % max(1, c["kv"] // 2)) for b in range(B)])
    shared = lens * 7 // 8 // P
    ends = np.cumsum(shared + K * (blocks - shared))
    n_pages, begin = int(ends[-1]), _ints(ends - shared - K * (blocks - shared)).repeat_interleave(K)[:, None]
    lens, shared = (_ints(v).repeat_interleave(K) for v in (lens, shared))
    used, shared = (lens + P - 1) // P, shared[:, None]
    at, beam = torch.arange(blocks, device=DEV)[None], torch.arange(R, device=DEV)
    place = begin + torch.where(at < shared, at, at + (beam % K)[:, None] * (blocks - shared))
    table = torch.where(at < used[:, None], r.perm(n_pages)[place], torch.full_like(place, -1)).to(torch.int32)
    refs = torch.zeros(n_pages + 1, dtype=torch.int32, device=DEV)
    refs.scatter_add_(0, torch.where(table < 0, n_pages, table).long().reshape(-1),
                      torch.ones(R * blocks, dtype=torch.int32, device=DEV))
    s.update(blocks=blocks, pages=n_pages, first=torch.cat([refs[:n_pages], table.reshape(-1), lens]))
    s["state"] = s["first"].clone()
    s["parents"] = (beam // K * K + r.below(K, R)).to(torch.int32)
    s["src"], s["dst"] = (torch.zeros(R, dtype=torch.int32, device=DEV) for _ in range(2))
    s["status"] = torch.zeros(3, dtype=torch.int32, device=DEV)
    s["kc"], s["vc"] = (r.normal(c["layers"], n_pages, P, c["dim"], dtype=TYPES[c["type"]]) for _ in range(2))
    return s


# ---- one pass -------------------------------------------------------------

def run(s):
    return _RUN[s["case"]["kind"]](s)


_lib = None


def _native():
    global _lib
    if _lib is None:
        here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        pkg = os.path.join(here, "callaghandev.ml_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from cdml import native
        native.init(0)
        _lib = native
    return _lib


def _call(name, *args):
    """One entry of the C ABI on torch's current stream; tensors pass as pointers."""
    n = _native()
    a = [t.data_ptr() if isinstance(t, torch.Tensor) else t for t in args]
    n.check(getattr(n.lib(), name)(*a, torch.cuda.current_stream().cuda_stream))


def _workspace(s, name, *args):
    """The workspace that a program keeps beside its state, made on the first pass."""
    if "ws" not in s:
        n, size = _native(), ctypes.c_size_t(0)
        n.check(getattr(n.lib(), name)(*args, ctypes.byref(size)))
        s["ws"] = torch.empty(max(256, size.value), device=DEV, dtype=torch.uint8)
    return s["ws"], s["ws"].numel()


def _run_plan(s):
    c = s["case"]
    B, P, N = c["batch"], c["page"], c["pages"]
    s["state"].copy_(s["first"])  # every pass is the same step
    refs, table, kv = _tables(s["state"], N, s["blocks"], B)
    out = {"refs": refs, "table": table, "kv_len": kv, "cu": s["cu"], "slots": s["slots"],
           "positions": s["positions"], "status": s["status"]}
    if own:
        _call("cdml_paged_plan", refs, N, P, table, s["blocks"], kv, s["new"], B, s["rows"], s["cu"], s["slots"],
              s["positions"], s["status"])
        return out
    new, at = s["new"].long(), torch.arange(s["blocks"], device=DEV)[None]
    old, have = kv.long(), (kv.long() + P - 1) // P
    need = (old + new + P - 1) // P - have
    ends, pages = torch.cumsum(new, 0), torch.cumsum(need, 0)
    free = refs == 0
    rank = torch.cumsum(free, 0) - 1
    code = ((pages[-1] > rank[-1] + 1).long() + 2 * ((new < 0) | (old < 0) | (old + new > s["blocks"] * P)).any()
            + 4 * (ends[-1] > s["rows"]))
    ok = code == 0
    order = torch.argsort((~free).to(torch.int32), stable=True)
    fresh = order[((pages - need)[:, None] + at - have[:, None]).clamp(0, N - 1)].to(torch.int32)
    table.copy_(torch.where(ok & (at >= have[:, None]) & (at < (have + need)[:, None]), fresh, table))
    refs.copy_(torch.where(ok & free & (rank < pages[-1]), 1, refs))
    kv.copy_(torch.where(ok, old + new, old))
    s["cu"][1:] = torch.where(ok, ends, 0)
    row = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(ends, row, right=True).clamp(max=B - 1)
    pos = old[b] + row - (ends - new)[b]
    real = ok & (row < ends[-1])
    page = table.reshape(-1)[(b * s["blocks"] + (pos // P).clamp(0, s["blocks"] - 1))]
    s["slots"].copy_(torch.where(real, page * P + pos % P, -1))
    s["positions"].copy_(torch.where(real, pos, 0))
    s["status"].copy_(torch.stack([code, pages[-1], ends[-1]]))
    return out


def _run_append(s):
    c = s["case"]
    n = c["pages"] * c["page"]
    if own:
        _call("cdml_paged_append", s["k"], c["dim"], s["v"], c["dim"], s["kc"], s["vc"],
              _native().CACHE[c["type"]], s["slots"], c["rows"], c["pages"], c["page"], c["dim"])
    else:
        to = torch.where(s["slots"] < 0, n, s["slots"]).long()
        s["kc"][to] = s["k"].to(s["kc"].dtype)
        s["vc"][to] = s["v"].to(s["vc"].dtype)
    return [s["kc"][:n], s["vc"][:n]]


def _scale(c):
    return float(np.float32(1.0) / np.sqrt(np.float32(c["hd"])))


def _run_attn(s):
    c = s["case"]
    B, H, HK, hd, P = c["batch"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    rows, n, m = s["rows"], max(s["news"]), max(s["lens"])
    if own:
        size = (rows, B, n, m, H, HK, hd)
        ws = _workspace(s, "cdml_paged_attn_workspace_size", *size)
        _call("cdml_paged_attn", s["q"], H * hd, s["kc"], s["vc"], _native().CACHE[c["type"]], s["pages"], P,
              s["table"], s["blocks"], s["kv_len"], s["cu"], s["o"], H * hd, *size, _scale(c), s["bad"], *ws)
        return s["o"]
    at = torch.arange(m, device=DEV)
    slot = (s["table"].long()[:, at // P] * P + at % P)                          # [B, m]
    key = s["kc"].view(-1, HK, hd)[slot].float().permute(0, 2, 3, 1)             # [B, HK, hd, m]
    val = s["vc"].view(-1, HK, hd)[slot].float().permute(0, 2, 1, 3)             # [B, HK, m, hd]
    i, first, length = torch.arange(n, device=DEV), s["cu"][:-1].long(), s["kv_len"].long()
    new = s["cu"][1:].long() - first
    row = (first[:, None] + i).clamp(max=rows - 1)                               # [B, n]
    q = s["q"].view(-1, HK, H // HK, hd)[row].permute(0, 2, 3, 1, 4).reshape(B, HK, -1, hd) * _scale(c)
    limit = (length - new)[:, None] + i                                          # last visible key
    seen = (at <= limit[:, :, None]) & (at < length[:, None, None])              # [B, n, m]
    score = torch.matmul(q, key.contiguous()).view(B, HK, H // HK, n, m)
    score.masked_fill_(~seen[:, None, None], -INF)
    score -= score.amax(-1, keepdim=True).clamp(min=-3e38)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(B, HK, -1, m), val.contiguous()).view(B, HK, H // HK, n, hd)
    out = (out / torch.where(total > 0, total, 1)).permute(0, 3, 1, 2, 4).reshape(B, n, H * hd)
    at_row = torch.arange(sum(s["news"]), device=DEV)
    b = torch.searchsorted(s["cu"][1:].long(), at_row, right=True)
    s["o"][:len(at_row)] = out[b, at_row - first[b]]
    return s["o"]


EOS = 2


def _alpha(c):
    return float(np.float32(c["alpha"]))


def _run_beam(s):
    c, o = s["case"], s["out"]
    B, K, V = c["batch"], c["beams"], c["vocab"]
    if own:
        ws = _workspace(s, "cdml_beam_select_workspace_size", B, K, V)
        _call("cdml_beam_select", s["x"], V, s["score"], s["len"], s["done"], B, K, V, EOS, c["alpha"], o["score"],
              o["len"], o["done"], o["parent"], o["token"], *ws)
        return o
    # in 64 bits: totals of different beams lie next to each other
    x, score, done = s["x"].double(), s["score"].double()[:, None], s["done"].bool()[:, None]
    top = x.amax(-1, keepdim=True)
    total = score + x - (top + (x - top).exp().sum(-1, keepdim=True).log())
    token = torch.arange(V, device=DEV)[None]
    total = torch.where(done, torch.where(token == EOS, score, -INF), total)
    length = s["len"].long()[:, None] + ~done
    key = (total / length.double().pow(_alpha(c))).view(B, K * V)
    best = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :K]
    parent = torch.arange(B, device=DEV)[:, None] * K + best // V
    picked = (best % V).reshape(-1)
    parent = parent.reshape(-1)
    o["score"].copy_(total.view(B, K * V).gather(1, best).reshape(-1))
    o["len"].copy_(length[parent, 0])
    o["done"].copy_(done[parent, 0] | (picked == EOS))
    o["parent"].copy_(parent)
    o["token"].copy_(picked)
    return o


def _run_reorder(s):
    c = s["case"]
    R, P, N, blocks = c["batch"] * c["beams"], c["page"], s["pages"], s["blocks"]
    s["state"].copy_(s["first"])  # every pass is the same step
    refs, table, kv = _tables(s["state"], N, blocks, R)
    out = {"refs": refs, "table": table, "kv_len": kv, "src": s["src"], "dst": s["dst"], "status": s["status"],
           "k": s["kc"], "v": s["vc"]}
    if own:
        ws = _workspace(s, "cdml_paged_reorder_workspace_size", R, blocks)
        _call("cdml_paged_reorder", refs, N, P, table, blocks, kv, s["parents"], R, s["src"], s["dst"], s["status"],
              *ws)
        _call("cdml_paged_copy", s["kc"], s["vc"], _native().CACHE[c["type"]], c["layers"], N * P * c["dim"], N, P,
              c["dim"], s["src"], s["dst"], kv, R)
        return out
    at, row = torch.arange(blocks, device=DEV)[None], torch.arange(R, device=DEV)
    old, length, parent = table.clone(), kv.long(), s["parents"].long()
    mine, full, open_ = length[parent], length[parent] // P, length[parent] % P > 0
    child = torch.full((R,), R, device=DEV).scatter_reduce_(0, parent, row, "amin")
    keeps = open_ & (child[parent] == row)
    taken, given = at < ((length + P - 1) // P)[:, None], at < (full + keeps)[:, None]
    ones = torch.ones(R * blocks, dtype=torch.int32, device=DEV)
    shared = old[parent]
    spare = torch.cat([refs, refs.new_zeros(1)])
    spare.scatter_add_(0, torch.where(taken, old, N).long().reshape(-1), -ones)
    spare.scatter_add_(0, torch.where(given, shared, N).long().reshape(-1), ones)
    copies = open_ & ~keeps
    turn = torch.cumsum(copies, 0) - 1
    free = spare[:N] == 0
    rank = torch.cumsum(free, 0) - 1
    page = torch.argsort((~free).to(torch.int32), stable=True)[turn.clamp(0, N - 1)].to(torch.int32)
    gets = copies & (turn <= rank[-1])
    refs.copy_(torch.where(free & (rank < gets.sum()), 1, spare[:N]))
    table.copy_(torch.where(given, shared, torch.where(gets[:, None] & (at == full[:, None]), page[:, None], old)))
    kv.copy_(torch.where(copies & ~gets, full * P, mine))
    s["src"].copy_(torch.where(gets, shared.gather(1, full.clamp(max=blocks - 1)[:, None])[:, 0], -1))
    s["dst"].copy_(torch.where(gets, page, -1))
    s["status"].copy_(torch.stack([(copies & ~gets).sum(), gets.sum(), torch.zeros_like(turn[0])]))
    # the copied tokens of every layer; a row without a copy writes a page's own first token to itself
    held = (torch.arange(P, device=DEV)[None] < (kv.long() % P)[:, None]) & gets[:, None]
    here = torch.where(gets, page.long(), page.long()[0])
    src = torch.where(gets, s["src"].long(), here)
    for_k, for_v = s["kc"][:, src], s["vc"][:, src]
    mask = held[None, :, :, None]
    to = torch.where(gets, here, N)
    _put(s["kc"], to, for_k, mask, here, N)
    _put(s["vc"], to, for_v, mask, here, N)
    return out


def _put(cache, to, tokens, mask, here, n):
    """cache[:, to] = tokens where mask, rows of `to` at n left out."""
    tokens = torch.where(mask, tokens, cache[:, here])
    wide = torch.cat([cache, cache[:, :1]], 1)
    wide[:, to] = tokens
    cache.copy_(wide[:, :n])


_RUN = {"plan": _run_plan, "append": _run_append, "attn": _run_attn, "beam": _run_beam, "reorder": _run_reorder}


# ---- the same results in float64 --------------------------------------------

def exact(case, seed):
    c, k = case, case["kind"]
    if k == "attn":
        s = prepare(case, seed)
        H, HK, hd, P = c["heads"], c["kv_heads"], c["hd"], c["page"]
        out, first = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), 0
        pairs = sum(n * m for m, n in zip(s["lens"], s["news"])) * H * hd
        if pairs > 3e11:
            return None
        for b, (m, n) in enumerate(zip(s["lens"], s["news"])):
            if not n:
                continue
            slot = s["table"][b].long().repeat_interleave(P)[:m] * P + torch.arange(m, device=DEV) % P
            hidden = torch.arange(m, device=DEV)[None] > torch.arange(m - n, m, device=DEV)[:, None]
            for h in range(H):
                at = slice(h // (H // HK) * hd, (h // (H // HK) + 1) * hd)
                q = s["q"][first:first + n, h * hd:(h + 1) * hd].double()
                w = (q @ s["kc"][slot, at].double().T.contiguous()) * _scale(c)
                w = torch.softmax(w.masked_fill(hidden, -INF), 1)
                out[first:first + n, h * hd:(h + 1) * hd] = w @ s["vc"][slot, at].double()
            first += n
        return out
    if k == "beam":
        s = prepare(case, seed)
        B, K, V = c["batch"], c["beams"], c["vocab"]
        score, done = s["score"].double().cpu().numpy(), s["done"].cpu().numpy()
        length = s["len"].cpu().numpy()
        logp = torch.log_softmax(s["x"].double(), 1)
        kept, at = torch.topk(logp, min(K, V), 1)
        kept, at = kept.cpu().numpy(), at.cpu().numpy()
        out = np.zeros(B * K)
        for b in range(B):
            found = []
            for r in range(b * K, (b + 1) * K):
                if done[r]:
                    found.append((score[r] / float(length[r]) ** _alpha(c), score[r]))
                else:
                    found += [((score[r] + p) / float(length[r] + 1) ** _alpha(c), score[r] + p) for p in kept[r]]
            found.sort(key=lambda f: -f[0])
            out[b * K:(b + 1) * K] = [f[1] for f in found[:K]]
        return {"score": out, "len": None, "done": None, "parent": None, "token": None}
    if k == "append":
        s = prepare(case, seed)
        n, at = c["pages"] * c["page"], s["slots"].long().cpu().numpy()
        out = []
        for new in (s["k"], s["v"]):
            cache = np.zeros((n, c["dim"]))
            cache[at[at >= 0]] = new.to(TYPES[c["type"]]).double().cpu().numpy()[at >= 0]
            out.append(cache)
        return out
    if k == "reorder":
        s = prepare(case, seed)
        P = c["page"]
        refs, table, kv = (t.cpu().numpy() for t in _tables(s["state"], s["pages"], s["blocks"], c["batch"] * c["beams"]))
        parents, refs, old, seen, waits = s["parents"].cpu().numpy(), refs.copy(), table.copy(), set(), []
        for r, n in enumerate(kv):
            np.subtract.at(refs, old[r, :-(-n // P)], 1)
        for r, p in enumerate(parents):
            np.add.at(refs, old[p, :kv[p] // P], 1)
            if kv[p] % P and p in seen:
                waits.append(p)
            elif kv[p] % P:
                refs[old[p, kv[p] // P]] += 1
            seen.add(p)
        k_out, v_out = s["kc"].double(), s["vc"].double()
        for p, page in zip(waits, np.flatnonzero(refs == 0)):
            src, n = int(old[p, kv[p] // P]), int(kv[p] % P)
            for out, cache in ((k_out, s["kc"]), (v_out, s["vc"])):
                out[:, int(page), :n] = cache[:, src, :n].double()
        return {"refs": None, "table": None, "kv_len": None, "src": None, "dst": None, "status": None,
                "k": k_out, "v": v_out}
    return None
