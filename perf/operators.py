"""Timing cases of the operators of a decode layer's step at reduced precision, in a plain form and as the package's kernels.

Four kinds of case:

  append   raw key and value rows of a ragged batch of prompt pieces into a paged cache of 16- or 8-bit rows, the keys
           normed and rotated on the way (KVCache.append), and the stored rows back (KVCache.gather)
  decode   attention of one new token of each sequence over such a cache (KVCache.attn_decode)
  step     the same from the raw projections: norms, rotation, append and attention (KVCache.full_core), and the new rows
  norm     the residual's addition, the layer norm and its 8-bit form for the projections (Context.add_rms_norm)

With `own` false, `run` computes them with elementary torch operations.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG_DIR = os.path.join(ROOT, "qwen3.8_27b_in_rust_amd")

HEADS, KV_HEADS, GROUP, DIM = 24, 4, 6, 256
Q_DIM, KV_DIM, QG_DIM = HEADS * DIM, KV_HEADS * DIM, 2 * HEADS * DIM
PAGE, LAYER = 16, 3
HIDDEN, FFN = 5120, 17408
EPS = 1e-6
# ggml type ids of a cache's rows
F32, F16, BF16, Q8_K = 0, 1, 30, 15
TYPES = {"f16": F16, "bf16": BF16, "q8_k": Q8_K}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
ROW_BYTES = {"f16": 2 * KV_DIM, "bf16": 2 * KV_DIM, "q8_k": KV_DIM + 4 * KV_HEADS}


def listed():
    return [
        # a whole prompt at once, into 8-bit rows
        {"name": "append_4096_q8k", "kind": "append", "type": "q8_k", "seqs": 1, "tokens": 4096, "base": 0},
        # the next pieces of twelve prompts, ragged and at positions inside pages
        {"name": "append_ragged_bf16", "kind": "append", "type": "bf16", "seqs": 12, "tokens": 1531, "base": 20011},
        # a few drafted tokens of two sequences: latency counts
        {"name": "append_6_f16", "kind": "append", "type": "f16", "seqs": 2, "tokens": 6, "base": 777},
        # a chat's decode step early in its context: two short launches, latency counts
        {"name": "step_1k_bf16", "kind": "step", "type": "bf16", "seqs": 1, "ctx": 1021},
        # the decode step of a long document, 16-bit and 8-bit rows
        {"name": "decode_32k_bf16", "kind": "decode", "type": "bf16", "seqs": 1, "ctx": 32768},
        {"name": "step_32k_q8k", "kind": "step", "type": "q8_k", "seqs": 1, "ctx": 32768},
        # the longest context of the 64-layer workload
        {"name": "decode_128k_q8k", "kind": "decode", "type": "q8_k", "seqs": 1, "ctx": 131072},
        # a server's step: 16 sequences of ragged lengths, the longest 32K
        {"name": "decode_batch16_f16", "kind": "decode", "type": "f16", "seqs": 16, "ctx": 32768},
        # a layer's input for one token, for a few (a draft verified), for a whole prompt, and a wide ragged one
        {"name": "norm_1", "kind": "norm", "tokens": 1, "width": HIDDEN},
        {"name": "norm_6", "kind": "norm", "tokens": 6, "width": HIDDEN},
        {"name": "norm_4096", "kind": "norm", "tokens": 4096, "width": HIDDEN},
        {"name": "norm_509_wide", "kind": "norm", "tokens": 509, "width": FFN},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "step", "norm"))
    if kind == "norm":
        width = rng.choice((HIDDEN, Q_DIM, FFN, 256 * rng.randint(1, 68)))
        return {"kind": kind, "tokens": _log_int(rng, 1, 4096 * HIDDEN // max(HIDDEN, width)), "width": width}
    case = {"kind": kind, "type": rng.choice(sorted(TYPES)), "seqs": _log_int(rng, 1, 16)}
    if kind == "append":
        return dict(case, tokens=_log_int(rng, case["seqs"], 4096), base=rng.choice((0, _log_int(rng, 1, 32768))))
    return dict(case, ctx=_log_int(rng, 1, 32768))


# ------------------------------------------------------------------ the program's side

_held = {}


def _pkg():
    if "q38amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location("q38amd", os.path.join(PKG_DIR, "__init__.py"),
                                                      submodule_search_locations=[PKG_DIR])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["q38amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["q38amd"]


def _ctx():
    """The program's one context."""
    if "ctx" not in _held:
        _held["ctx"] = _pkg().Context(0)
    return _held["ctx"]


class _State:
    """Buffers of one case; the cache is given back with it."""

    def __init__(self, case):
        self.case, self.kv = case, None

    def __del__(self):
        if self.kv is not None:
            self.kv.close()


class _Gen:
    """Seeded device tensors."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) * 7919 + 29)

    def normal(self, *shape, sigma=1.0, mean=0.0):
        x = torch.randn(shape, generator=self.g, device="cuda", dtype=torch.float32)
        return x.mul_(sigma).add_(mean) if (sigma, mean) != (1.0, 0.0) else x

    def permutation(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _lengths(n, most):
    """Ragged lengths of n sequences: the longest, then down to a sixteenth of it, evenly over the logarithm."""
    return [max(1, int(most * 16.0 ** (-i / max(1, n - 1)))) for i in range(n)]


def _pieces(case):
    """(first position, tokens) of each sequence's piece: the tokens in ragged shares, later sequences further on."""
    n, total = case["seqs"], case["tokens"]
    shares = _lengths(n, 1 << 20)
    counts = [max(1, total * s // sum(shares)) for s in shares]
    counts[0] += max(0, total - sum(counts))
    return [(case["base"] + (37 * i if case["base"] else 0), c) for i, c in enumerate(counts)]


def _angles(positions):
    """The rotation's angles [n][32] of positions: the position times the scale, product by product in 32 bits, as the model defines them."""
    scale = np.float32(np.float32(10000000.0) ** np.float32(-2.0 / 64.0))
    theta, rows = np.array(positions, np.float32), []
    for _ in range(32):
        rows.append(theta)
        theta = (theta * scale).astype(np.float32)
    return torch.from_numpy(np.stack(rows, 1)).cuda()


def _inputs(case, g):
    """A case's inputs, in the order that they are drawn."""
    kind, x = case["kind"], {}
    if kind == "norm":
        n, w = case["tokens"], case["width"]
        # the residual stream of a deep layer is larger than what a layer adds, with a few large channels
        x["residual"] = g.normal(n, w, sigma=3.0) * (1.0 + 20.0 * (g.normal(1, w) > 2.5))
        x["x"] = g.normal(n, w, sigma=0.7)
        x["weight"] = g.normal(w, sigma=0.1, mean=1.0)
        return x
    if kind == "append":
        n = sum(c for _, c in _pieces(case))
        return {"k_norm": g.normal(DIM, sigma=0.1, mean=1.0), "key": g.normal(n, KV_DIM), "value": g.normal(n, KV_DIM)}
    n = case["seqs"]
    if kind == "decode":
        x = {"q": g.normal(n, Q_DIM), "gate": g.normal(n, Q_DIM)}
    else:
        x = {"q_norm": g.normal(DIM, sigma=0.1, mean=1.0), "k_norm": g.normal(DIM, sigma=0.1, mean=1.0),
             "qg": g.normal(n, QG_DIM), "key": g.normal(n, KV_DIM), "value": g.normal(n, KV_DIM)}
    total = sum(_lengths(n, case["ctx"]))
    return dict(x, k=g.normal(total, KV_DIM), v=g.normal(total, KV_DIM))


def _page_lists(case, g):
    """Each sequence's pages in a shared pool, in a random order, as a program that serves many requests has them."""
    ends = [b + c for b, c in _pieces(case)] if case["kind"] == "append" else _lengths(case["seqs"], case["ctx"])
    counts = [-(-e // PAGE) for e in ends]
    order, at, lists = g.permutation(sum(counts)).tolist(), 0, []
    for c in counts:
        lists.append(order[at:at + c])
        at += c
    return lists


def _cached_rows(case):
    """(sequence, position) of each row that the cache holds beforehand, or that an append brings."""
    spans = _pieces(case) if case["kind"] == "append" else [(0, c) for c in _lengths(case["seqs"], case["ctx"])]
    return (np.concatenate([np.full(c, i) for i, (_, c) in enumerate(spans)]),
            np.concatenate([np.arange(b, b + c) for b, c in spans]))


def prepare(case, seed):
    g, s = _Gen(seed), _State(case)
    s.x = _inputs(case, g)
    new = lambda *shape, dtype=torch.float32: torch.zeros(shape, device="cuda", dtype=dtype)  # noqa: E731
    if case["kind"] == "norm":
        if own:
            n, w = case["tokens"], case["width"]
            s.h, s.y, s.values = new(n, w), new(n, w), new(n, w)
            s.q8k = new(_ctx().q8k_bytes(n, w), dtype=torch.uint8)
        torch.cuda.synchronize()
        return s
    lists = _page_lists(case, g)
    seq, pos = _cached_rows(case)
    if case["kind"] == "append":
        s.spans = _pieces(case)
    else:
        s.positions = [c - 1 for c in _lengths(case["seqs"], case["ctx"])]
    if own:
        _prepare_own(s, lists, new)
    else:
        _prepare_plain(s, lists, seq, pos, new)
    torch.cuda.synchronize()
    return s


def _prepare_own(s, lists, new):
    case, ctx = s.case, _ctx()
    s.kv = _pkg().KVCache(ctx, n_slots=1, max_pages=sum(map(len, lists)), max_seqs=len(lists),
                          max_tokens_per_seq=PAGE * max(map(len, lists)), ggml_type=TYPES[case["type"]])
    s.seqs = [s.kv.seq_create() for _ in lists]
    for q, pages in zip(s.seqs, lists):
        s.kv.seq_set_pages(q, pages)
    if case["kind"] == "append":
        n = sum(c for _, c in s.spans)
    else:
        n = case["seqs"]
        s.out = new(n, Q_DIM)
        torch.cuda.synchronize()
        at = 0
        for q, p in zip(s.seqs, s.positions):
            s.kv.write(LAYER, q, 0, p + 1, s.x["k"][at:].data_ptr(), s.x["v"][at:].data_ptr())
            at += p + 1
        ctx.sync()
        del s.x["k"], s.x["v"]
    dtype = DTYPES.get(case["type"], torch.float32)
    s.k, s.v = new(n, KV_DIM, dtype=dtype), new(n, KV_DIM, dtype=dtype)


def _prepare_plain(s, lists, seq, pos, new):
    case = s.case
    table = np.zeros((len(lists), max(map(len, lists))), np.int64)
    for i, pages in enumerate(lists):
        table[i, :len(pages)] = pages
    s.table = torch.from_numpy(table).cuda()
    n_rows = PAGE * sum(map(len, lists))
    if case["type"] == "q8_k":
        s.pool = [(new(n_rows, KV_HEADS, DIM, dtype=torch.int8), new(n_rows, KV_HEADS)) for _ in range(2)]
    else:
        s.pool = [(new(n_rows, KV_HEADS, DIM, dtype=DTYPES[case["type"]]),) for _ in range(2)]
    if case["kind"] == "append":
        s.at = torch.from_numpy(table[seq, pos // PAGE] * PAGE + pos % PAGE).cuda()
        s.theta = _angles(pos)
        return
    at = torch.from_numpy(table[seq, pos // PAGE] * PAGE + pos % PAGE).cuda()
    for pool, name in zip(s.pool, ("k", "v")):
        _store(pool, at, s.x.pop(name).view(-1, KV_HEADS, DIM))
    last = np.array(s.positions)
    s.last = torch.from_numpy(last).cuda()
    s.at = torch.from_numpy(table[np.arange(len(lists)), last // PAGE] * PAGE + last % PAGE).cuda()
    s.theta = _angles(last)


# ------------------------------------------------------------------ the plain forms


def _rms_scale(x):
    """1 / sqrt(mean of squares + eps) of the rows, the mean and each later step rounded to 32 bits."""
    mean = (x.double().square().sum(-1, keepdim=True) / x.shape[-1]).float()
    root = torch.sqrt((mean + EPS).double()).float()
    return (1.0 / root.double()).float()


def _rms(x, w):
    return x * _rms_scale(x) * w


def _rope(x, theta):
    """x [n][heads][256]: pairs (p, p + 32), p < 32, turned by theta [n][32]."""
    c, s = torch.cos(theta)[:, None, :], torch.sin(theta)[:, None, :]
    a, b = x[..., :32], x[..., 32:64]
    return torch.cat((a * c - b * s, a * s + b * c, x[..., 64:]), -1)


def _q8k(x):
    """8-bit quants and scale of rows of 256: the first value of largest size becomes -127."""
    m = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    inverse = torch.where(m == 0, 0.0, (-127.0 / m.double()).float())
    scale = torch.where(m == 0, 0.0, (1.0 / inverse.double()).float())
    return torch.round(x * inverse).clamp_max(127.0).to(torch.int8), scale[..., 0]


def _store(pool, at, rows):
    if len(pool) == 2:
        pool[0][at], pool[1][at] = _q8k(rows)
    else:
        pool[0][at] = rows.to(pool[0].dtype)


def _load(pool, at):
    """Rows as the 32-bit values that they stand for."""
    return pool[0][at].float() * pool[1][at][..., None] if len(pool) == 2 else pool[0][at].float()


def _stored(pool, at):
    """Rows in the cache's 16-bit type, or the values that its 8-bit rows stand for."""
    return (_load(pool, at) if len(pool) == 2 else pool[0][at]).reshape(-1, KV_DIM)


def _attend(s, q, gate):
    """q, gate [n][24][256]: each sequence's rows by its page table, padded to the longest and masked past its last position."""
    n, length = s.table.shape[0], s.table.shape[1] * PAGE
    at = (s.table[:, :, None] * PAGE + torch.arange(PAGE, device="cuda")).view(n, length)
    k = _load(s.pool[0], at).permute(0, 2, 3, 1).contiguous()  # [n][4][256][length]
    x = torch.matmul(q.view(n, KV_HEADS, GROUP, DIM), k) / 16.0
    del k
    late = torch.arange(length, device="cuda")[None, :] > s.last[:, None]
    x.masked_fill_(late[:, None, None, :], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    v = _load(s.pool[1], at).permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return (o.reshape(n, HEADS, DIM) / (1.0 + torch.exp(-gate))).view(n, Q_DIM)


def run(s):
    if own:
        return _run_own(s)
    kind, x = s.case["kind"], s.x
    if kind == "norm":
        h = x["x"] + x["residual"]
        y = _rms(h, x["weight"])
        q, scale = _q8k(y.view(h.shape[0], -1, 256))
        return {"h": h, "y": y, "q8k": (q.float() * scale[..., None]).view_as(h)}
    if kind == "append":
        k = _rope(_rms(x["key"].view(-1, KV_HEADS, DIM), x["k_norm"]), s.theta)
        _store(s.pool[0], s.at, k)
        _store(s.pool[1], s.at, x["value"].view(-1, KV_HEADS, DIM))
        return {"k": _stored(s.pool[0], s.at), "v": _stored(s.pool[1], s.at)}
    if kind == "decode":
        return {"out": _attend(s, x["q"].view(-1, HEADS, DIM), x["gate"].view(-1, HEADS, DIM))}
    qg = x["qg"].view(-1, HEADS, 2, DIM)
    q = _rope(_rms(qg[:, :, 0], x["q_norm"]), s.theta)
    k = _rope(_rms(x["key"].view(-1, KV_HEADS, DIM), x["k_norm"]), s.theta)
    _store(s.pool[0], s.at, k)
    _store(s.pool[1], s.at, x["value"].view(-1, KV_HEADS, DIM))
    return {"out": _attend(s, q, qg[:, :, 1]), "k": _stored(s.pool[0], s.at), "v": _stored(s.pool[1], s.at)}


# ------------------------------------------------------------------ the package's calls


def _gather(s, first, counts):
    ty = TYPES[s.case["type"]]
    s.kv.gather(LAYER, s.seqs, first, counts, s.k.data_ptr(), s.v.data_ptr(), ggml_type=F32 if ty == Q8_K else ty)
    return {"k": s.k, "v": s.v}


def _run_own(s):
    ctx, case = _ctx(), s.case
    kind, p = case["kind"], {k: v.data_ptr() for k, v in s.x.items()}
    if kind == "norm":
        n, w = case["tokens"], case["width"]
        ctx.add_rms_norm(n, w, p["x"], p["weight"], residual=p["residual"], sum_out=s.h.data_ptr(), y=s.y.data_ptr(),
                         q8k=s.q8k.data_ptr())
        ctx.dequantize_q8_k(n, w, s.q8k.data_ptr(), s.values.data_ptr())
        return {"h": s.h, "y": s.y, "q8k": s.values}
    if kind == "append":
        first, counts = [b for b, _ in s.spans], [c for _, c in s.spans]
        s.kv.append(LAYER, s.seqs, first, counts, p["k_norm"], p["key"], p["value"])
        return _gather(s, first, counts)
    if kind == "decode":
        s.kv.attn_decode(LAYER, s.seqs, s.positions, p["q"], s.out.data_ptr(), gate=p["gate"])
        return {"out": s.out}
    s.kv.full_core(LAYER, s.seqs, s.positions, p["q_norm"], p["k_norm"], p["qg"], p["key"], p["value"], s.out.data_ptr())
    return dict(_gather(s, s.positions, [1] * len(s.seqs)), out=s.out)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    kind = case["kind"]
    if kind == "norm":
        # both inputs and the weight read; h, y and the 8-bit row written, and that row read and written as values
        n = case["tokens"] * case["width"]
        return {"bytes": 16 * n + 4 * case["width"] + n // 256 * (292 + 260) + 4 * n, "flops": 8 * n}
    row = ROW_BYTES[case["type"]]
    back = 4 * KV_DIM if case["type"] == "q8_k" else row
    if kind == "append":
        n = sum(c for _, c in _pieces(case))
        return {"bytes": 2 * n * (4 * KV_DIM + 2 * row + back), "flops": 10 * n * KV_DIM}
    n, cached = case["seqs"], sum(_lengths(case["seqs"], case["ctx"]))
    b, f = 2 * cached * row, cached * HEADS * DIM * 4
    if kind == "decode":
        return {"bytes": b + 12 * n * Q_DIM, "flops": f}
    return {"bytes": b + 4 * n * (QG_DIM + 2 * KV_DIM + Q_DIM) + 2 * n * (row + back), "flops": f}


# ------------------------------------------------------------------ the same in 64 bits


def _rounded(x, ty):
    """Cached rows [n][4][256] as the 64-bit numbers that their type holds."""
    if ty != "q8_k":
        return x.to(DTYPES[ty]).double()
    m = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    inverse = torch.where(m == 0, 0.0, torch.tensor(-127.0, device=x.device) / m)
    codes = torch.clamp(torch.round(inverse * x), max=127.0)
    return codes.double() * torch.where(m == 0, 0.0, torch.reciprocal(inverse)).double()


def _turned64(x, w, positions):
    """Normed rows [n][heads][256] in 64 bits, turned by their positions' angles (as a complex product)."""
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    turn = torch.polar(torch.ones_like(t := _angles(positions).double()), t)[:, None, :]
    z = torch.complex(x[..., :32], x[..., 32:64]) * turn
    return torch.cat((z.real, z.imag, x[..., 64:]), -1)


def exact(case, seed):
    x, kind = _inputs(case, _Gen(seed)), case["kind"]
    if kind == "norm":
        h = x["x"].double() + x["residual"].double()
        # 8-bit values are whole steps of a scale: no 64-bit value stands for them
        return {"h": h, "y": h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * x["weight"].double(), "q8k": None}
    ty = case["type"]
    if kind == "append":
        if ty == "q8_k":
            return None
        k = _turned64(x["key"].view(-1, KV_HEADS, DIM), x["k_norm"], _cached_rows(case)[1])
        return {"k": k.reshape(-1, KV_DIM), "v": x["value"].double()}
    lengths, at, out, news = _lengths(case["seqs"], case["ctx"]), 0, [], None
    if kind == "decode":
        q, gate = (x[n].double().view(-1, HEADS, DIM) for n in ("q", "gate"))
    else:
        last = [c - 1 for c in lengths]
        qg = x["qg"].view(-1, HEADS, 2, DIM)
        q, gate = _turned64(qg[:, :, 0], x["q_norm"], last), qg[:, :, 1].double()
        k_new = _turned64(x["key"].view(-1, KV_HEADS, DIM), x["k_norm"], last)
        news = {"k": k_new.reshape(-1, KV_DIM), "v": x["value"].double()}
    for i, c in enumerate(lengths):
        k, v = (x[n][at:at + c].view(-1, KV_HEADS, DIM) for n in ("k", "v"))
        at += c
        if news:
            # the token's own rows take the last position, in the cache's type
            k = torch.cat((k[:-1], k_new[i:i + 1].float()))
            v = torch.cat((v[:-1], x["value"][i:i + 1].view(1, KV_HEADS, DIM)))
        k, v = _rounded(k, ty), _rounded(v, ty)
        for h in range(HEADS):
            p = torch.softmax(k[:, h // GROUP].contiguous() @ q[i, h] / 16.0, 0)
            out.append(p @ v[:, h // GROUP].contiguous() * torch.sigmoid(gate[i, h]))
    out = torch.stack(out).view(-1, Q_DIM)
    if not news:
        return {"out": out}
    return dict(news, out=out) if ty != "q8_k" else {"out": out, "k": None, "v": None}
