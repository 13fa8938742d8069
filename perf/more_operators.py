"""Timing cases of long contexts in little memory, in a plain form and as the package's kernels.

Six kinds of case, over a paged cache:

  append   raw key and value rows of a ragged batch into 4-bit rows, the keys normed and rotated on the way
           (KVCache.append), and the values that the stored rows stand for (KVCache.gather)
  decode   attention of one new token of each sequence over 4-bit rows (KVCache.attn_decode)
  step     the same from the raw projections: norms, rotation, append and attention (KVCache.full_core), and the new rows
  weigh    the same attention over rows of any type, adding up the weight that each cached token gets
           (KVCache.track_weights, KVCache.attn_decode), and the sums (KVCache.weights_get)
  observe  the weights that a prompt's last tokens give to all before them, added to those sums (KVCache.attn_observe)
  evict    each kv head's tokens of least weight out of the cache, the rows that stay moved together (KVCache.evict)

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
PAGE, LAYER, BLOCK = 16, 3, 32
EPS = 1e-6
# ggml type ids of a cache's rows
F32, F16, BF16, Q8_K, MXFP4 = 0, 1, 30, 15, 39
TYPES = {"f16": F16, "bf16": BF16, "q8_k": Q8_K, "mxfp4": MXFP4}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
ROW_BYTES = {"f16": 2 * KV_DIM, "bf16": 2 * KV_DIM, "q8_k": KV_DIM + 4 * KV_HEADS, "mxfp4": KV_DIM // 2 + KV_DIM // BLOCK}


def listed():
    return [
        # a whole prompt at once
        {"name": "append_4096", "kind": "append", "type": "mxfp4", "seqs": 1, "tokens": 4096, "base": 0},
        # the next pieces of twelve prompts, ragged and at positions inside pages
        {"name": "append_ragged", "kind": "append", "type": "mxfp4", "seqs": 12, "tokens": 1531, "base": 20011},
        # a chat's decode step early in its context: latency counts
        {"name": "step_1k", "kind": "step", "type": "mxfp4", "seqs": 1, "ctx": 1021},
        # the decode step of a long document, and of the longest context of the 64-layer workload
        {"name": "decode_32k", "kind": "decode", "type": "mxfp4", "seqs": 1, "ctx": 32768},
        {"name": "decode_128k", "kind": "decode", "type": "mxfp4", "seqs": 1, "ctx": 131072},
        # a server's step: 16 sequences of ragged lengths, the longest 32K
        {"name": "decode_batch16", "kind": "decode", "type": "mxfp4", "seqs": 16, "ctx": 32768},
        # the decode step of a document whose cache is to be cut down, 16-bit rows, and of eight of them in 4 bits
        {"name": "weigh_32k_bf16", "kind": "weigh", "type": "bf16", "seqs": 1, "ctx": 32768},
        {"name": "weigh_batch8_mxfp4", "kind": "weigh", "type": "mxfp4", "seqs": 8, "ctx": 16384},
        # a prompt's last 32 tokens over all of it before the cache is cut down; the seven tokens of a short question
        {"name": "observe_32_of_32k_mxfp4", "kind": "observe", "type": "mxfp4", "tokens": 32, "ctx": 32768},
        {"name": "observe_7_of_1000_bf16", "kind": "observe", "type": "bf16", "tokens": 7, "ctx": 1000},
        # a long document down to a quarter, and a server's eight chats down to 60 per cent each
        {"name": "evict_32k_bf16", "kind": "evict", "type": "bf16", "seqs": 1, "ctx": 32768, "keep": 25, "recent": 128},
        {"name": "evict_batch8_q8k", "kind": "evict", "type": "q8_k", "seqs": 8, "ctx": 4003, "keep": 60, "recent": 61},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "step", "weigh", "observe", "evict"))
    if kind == "observe":
        ctx = _log_int(rng, 1, 32768)
        return {"kind": kind, "type": rng.choice(sorted(TYPES)), "tokens": _log_int(rng, 1, min(64, ctx)), "ctx": ctx}
    if kind == "append":
        seqs = _log_int(rng, 1, 16)
        return {"kind": kind, "type": "mxfp4", "seqs": seqs, "tokens": _log_int(rng, seqs, 4096),
                "base": rng.choice((0, _log_int(rng, 1, 32768)))}
    case = {"kind": kind, "type": "mxfp4", "seqs": _log_int(rng, 1, 16), "ctx": _log_int(rng, 1, 32768)}
    if kind in ("weigh", "evict"):
        case.update(type=rng.choice(sorted(TYPES)), seqs=_log_int(rng, 1, 8))
    if kind == "evict":
        case.update(ctx=_log_int(rng, 1, 16384), keep=rng.randint(5, 100), recent=_log_int(rng, 1, 256))
    return case


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
        self.g.manual_seed(int(seed) * 7919 + 31)

    def normal(self, *shape, sigma=1.0, mean=0.0):
        x = torch.randn(shape, generator=self.g, device="cuda", dtype=torch.float32)
        return x.mul_(sigma).add_(mean) if (sigma, mean) != (1.0, 0.0) else x

    def permutation(self, n):
        return torch.randperm(n, generator=self.g, device="cuda")


def _lengths(n, most):
    """Ragged lengths of n sequences: the longest, then down to a sixteenth of it, evenly over the logarithm."""
    return [max(1, int(most * 16.0 ** (-i / max(1, n - 1)))) for i in range(n)]


def _counts(case):
    """Tokens that each sequence holds before the call."""
    return _lengths(case.get("seqs", 1), case["ctx"])


def _kept(case):
    """(tokens to keep, of them the most recent) of each sequence."""
    keep = [max(1, c * case["keep"] // 100) for c in _counts(case)]
    return keep, [min(k, case["recent"]) for k in keep]


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
    if kind == "append":
        n = sum(c for _, c in _pieces(case))
        return {"k_norm": g.normal(DIM, sigma=0.1, mean=1.0), "key": g.normal(n, KV_DIM), "value": g.normal(n, KV_DIM)}
    counts = _counts(case)
    n, total = len(counts), sum(counts)
    if kind == "observe":
        x["q"] = g.normal(case["tokens"], Q_DIM)
    elif kind in ("decode", "weigh"):
        x = {"q": g.normal(n, Q_DIM), "gate": g.normal(n, Q_DIM)}
    elif kind == "step":
        x = {"q_norm": g.normal(DIM, sigma=0.1, mean=1.0), "k_norm": g.normal(DIM, sigma=0.1, mean=1.0),
             "qg": g.normal(n, QG_DIM), "key": g.normal(n, KV_DIM), "value": g.normal(n, KV_DIM)}
    else:
        # sums of softmax weights over many steps: a few tokens hold most, many next to nothing, some none at all
        w = torch.exp(g.normal(total, KV_HEADS, sigma=2.0, mean=-3.0))
        x["weights"] = w * (g.normal(total, KV_HEADS) > -1.5)
    return dict(x, k=g.normal(total, KV_DIM), v=g.normal(total, KV_DIM))


def _page_lists(case, g):
    """Each sequence's pages in a shared pool, in a random order, as a program that serves many requests has them."""
    ends = [b + c for b, c in _pieces(case)] if case["kind"] == "append" else _counts(case)
    counts = [-(-e // PAGE) for e in ends]
    order, at, lists = g.permutation(sum(counts)).tolist(), 0, []
    for c in counts:
        lists.append(order[at:at + c])
        at += c
    return lists


def _cached_rows(case):
    """(sequence, position) of each row that the cache holds beforehand, or that an append brings."""
    spans = _pieces(case) if case["kind"] == "append" else [(0, c) for c in _counts(case)]
    return (np.concatenate([np.full(c, i) for i, (_, c) in enumerate(spans)]),
            np.concatenate([np.arange(b, b + c) for b, c in spans]))


def prepare(case, seed):
    g, s = _Gen(seed), _State(case)
    s.x = _inputs(case, g)
    new = lambda *shape, dtype=torch.float32: torch.zeros(shape, device="cuda", dtype=dtype)  # noqa: E731
    s.lists = _page_lists(case, g)
    seq, pos = _cached_rows(case)
    if case["kind"] == "append":
        s.spans = _pieces(case)
    else:
        s.counts = _counts(case)
        s.positions = [c - 1 for c in s.counts]
    if own:
        _prepare_own(s, new)
    else:
        _prepare_plain(s, seq, pos, new)
    torch.cuda.synchronize()
    return s


def _prepare_own(s, new):
    case, ctx, lists = s.case, _ctx(), s.lists
    kind = case["kind"]
    s.kv = _pkg().KVCache(ctx, n_slots=1, max_pages=sum(map(len, lists)), max_seqs=len(lists),
                          max_tokens_per_seq=PAGE * max(map(len, lists)), ggml_type=TYPES[case["type"]])
    if kind in ("weigh", "observe", "evict"):
        s.kv.track_weights(True)
    s.seqs = [s.kv.seq_create() for _ in lists]
    for q, pages in zip(s.seqs, lists):
        s.kv.seq_set_pages(q, pages)
    dtype = DTYPES.get(case["type"], torch.float32)
    if kind == "append":
        n = sum(c for _, c in s.spans)
        s.k, s.v = new(n, KV_DIM), new(n, KV_DIM)
        return
    torch.cuda.synchronize()
    at = 0
    for q, c in zip(s.seqs, s.counts):
        s.kv.write(LAYER, q, 0, c, s.x["k"][at:].data_ptr(), s.x["v"][at:].data_ptr())
        at += c
    ctx.sync()
    del s.x["k"], s.x["v"]
    n, total = len(s.counts), sum(s.counts)
    if kind == "evict":
        kept = sum(_kept(case)[0])
        s.k, s.v = new(kept, KV_DIM, dtype=dtype), new(kept, KV_DIM, dtype=dtype)
        s.weights, s.tokens = new(kept, KV_HEADS), new(kept, KV_HEADS, dtype=torch.int32)
        return
    s.weights = new(total, KV_HEADS)
    s.out = new(n, Q_DIM)
    s.k, s.v = new(n, KV_DIM), new(n, KV_DIM)


def _prepare_plain(s, seq, pos, new):
    case, lists = s.case, s.lists
    table = np.zeros((len(lists), max(map(len, lists))), np.int64)
    for i, pages in enumerate(lists):
        table[i, :len(pages)] = pages
    s.table = torch.from_numpy(table).cuda()
    n_rows = PAGE * sum(map(len, lists))
    if case["type"] == "q8_k":
        s.pool = [(new(n_rows, KV_HEADS, DIM, dtype=torch.int8), new(n_rows, KV_HEADS)) for _ in range(2)]
    elif case["type"] == "mxfp4":
        s.pool = [(new(n_rows, KV_HEADS, DIM, dtype=torch.int8), new(n_rows, KV_HEADS, DIM // BLOCK, dtype=torch.int8))
                  for _ in range(2)]
    else:
        s.pool = [(new(n_rows, KV_HEADS, DIM, dtype=DTYPES[case["type"]]),) for _ in range(2)]
    at = torch.from_numpy(table[seq, pos // PAGE] * PAGE + pos % PAGE).cuda()
    if case["kind"] == "append":
        s.at, s.theta = at, _angles(pos)
        return
    for pool, name in zip(s.pool, ("k", "v")):
        _store(pool, at, s.x.pop(name).view(-1, KV_HEADS, DIM))
    s.rows_at = list(at.split(s.counts))
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


def _power(e):
    """2^e, exactly."""
    return torch.exp2(e.double()).float()


def _mxfp4(x):
    """Codes (sign times 0 .. 7 for 0, 0.5, 1, 1.5, 2, 3, 4, 6; halfway to the even code) and exponents of rows in blocks
    of 32: the scale is the smallest power of two of which the block's largest value has at most 7, within 2^-125 .. 2^125."""
    b = x.unflatten(-1, (-1, BLOCK))
    f, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    e = (e - 3 + (f > 0.875).to(e.dtype)).clamp(-125, 125)
    a = b.abs() * _power(-e)
    code = ((a > 0.25).to(torch.int8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.int8)
    return torch.where(b < 0, -code, code).flatten(-2), e[..., 0].to(torch.int8)


def _mxfp4_values(code, e):
    a = code.abs().float()
    a = torch.where(a <= 4, 0.5 * a, torch.where(a == 7, 6.0, a - 2.0))
    a = torch.where(code < 0, -a, a)
    return (a.unflatten(-1, (-1, BLOCK)) * _power(e)[..., None]).flatten(-2)


def _store(pool, at, rows):
    if len(pool) == 1:
        pool[0][at] = rows.to(pool[0].dtype)
    else:
        pool[0][at], pool[1][at] = _mxfp4(rows) if pool[1].dtype == torch.int8 else _q8k(rows)


def _load(pool, at):
    """Rows as the 32-bit values that they stand for."""
    if len(pool) == 1:
        return pool[0][at].float()
    if pool[1].dtype == torch.int8:
        return _mxfp4_values(pool[0][at], pool[1][at])
    return pool[0][at].float() * pool[1][at][..., None]


def _stored(pool, at):
    """Rows in the cache's 16-bit type, or the values that its 8- or 4-bit rows stand for."""
    return (pool[0][at] if len(pool) == 1 else _load(pool, at)).reshape(-1, KV_DIM)


def _attend(s, q, gate):
    """q, gate [n][24][256]: each sequence's rows by its page table, padded to the longest and masked past its last position.
    The gated outputs, and the softmax weights [n][4][6][length]."""
    n, length = s.table.shape[0], s.table.shape[1] * PAGE
    at = (s.table[:, :, None] * PAGE + torch.arange(PAGE, device="cuda")).view(n, length)
    k = _load(s.pool[0], at).permute(0, 2, 3, 1).contiguous()  # [n][4][256][length]
    x = torch.matmul(q.view(n, KV_HEADS, GROUP, DIM), k) / 16.0
    del k
    late = torch.arange(length, device="cuda")[None, :] > s.last[:, None]
    x.masked_fill_(late[:, None, None, :], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    v = _load(s.pool[1], at).permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p, v)
    return (o.reshape(n, HEADS, DIM) / (1.0 + torch.exp(-gate))).view(n, Q_DIM), p


def _observed(s, q):
    """Weights [tokens][4] that the last n tokens' queries [n][24][256] give, each over the positions up to its own."""
    n, length = q.shape[0], s.counts[0]
    k = _load(s.pool[0], s.rows_at[0]).permute(1, 2, 0).contiguous()  # [4][256][length]
    rows = q.view(n, KV_HEADS, GROUP, DIM).permute(1, 0, 2, 3).reshape(KV_HEADS, n * GROUP, DIM)
    x = torch.matmul(rows, k).view(KV_HEADS, n, GROUP, length) / 16.0
    last = torch.arange(length - n, length, device="cuda")
    x.masked_fill_((torch.arange(length, device="cuda")[None, :] > last[:, None])[None, :, None, :], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    return p.sum((1, 2)).t().contiguous()


def _evict(s):
    """Of each sequence and kv head: the recent tokens and those of most weight stay, the earlier of equal ones; the holes
    among the first positions take the later rows, both in order."""
    keep, recent = _kept(s.case)
    k, v, weights, tokens, w0 = [], [], [], [], 0
    for at, c, n, r in zip(s.rows_at, s.counts, keep, recent):
        w = s.x["weights"][w0:w0 + c]
        w0 += c
        rank = w.clone()
        rank[c - r:] = math.inf
        first = torch.sort(rank, dim=0, descending=True, stable=True).indices[:n]  # [n][4]
        stays = torch.zeros(c, KV_HEADS, device="cuda", dtype=torch.bool).scatter_(0, first, True)
        moved = torch.arange(n, device="cuda")[:, None].repeat(1, KV_HEADS)
        # in the order of heads, then positions, on both sides
        moved.t()[~stays[:n].t()] = n + stays[n:].t().nonzero()[:, 1]
        rows = at[moved]
        for pool in s.pool:
            got = [part[rows, torch.arange(KV_HEADS, device="cuda")] for part in pool]
            for part, x in zip(pool, got):
                part[at[:n]] = x
        k.append(_stored(s.pool[0], at[:n]))
        v.append(_stored(s.pool[1], at[:n]))
        weights.append(w.gather(0, moved))
        tokens.append(moved.int())
    return {"k": torch.cat(k), "v": torch.cat(v), "weights": torch.cat(weights), "tokens": torch.cat(tokens)}


def run(s):
    if own:
        return _run_own(s)
    kind, x = s.case["kind"], s.x
    if kind == "append":
        k = _rope(_rms(x["key"].view(-1, KV_HEADS, DIM), x["k_norm"]), s.theta)
        _store(s.pool[0], s.at, k)
        _store(s.pool[1], s.at, x["value"].view(-1, KV_HEADS, DIM))
        return {"k": _stored(s.pool[0], s.at), "v": _stored(s.pool[1], s.at)}
    if kind == "observe":
        return {"weights": _observed(s, x["q"].view(-1, HEADS, DIM))}
    if kind == "evict":
        return _evict(s)
    if kind != "step":
        out, p = _attend(s, x["q"].view(-1, HEADS, DIM), x["gate"].view(-1, HEADS, DIM))
        if kind == "decode":
            return {"out": out}
        p = p.sum(2)
        return {"out": out, "weights": torch.cat([p[i, :, :c].t() for i, c in enumerate(s.counts)])}
    qg = x["qg"].view(-1, HEADS, 2, DIM)
    q = _rope(_rms(qg[:, :, 0], x["q_norm"]), s.theta)
    k = _rope(_rms(x["key"].view(-1, KV_HEADS, DIM), x["k_norm"]), s.theta)
    _store(s.pool[0], s.at, k)
    _store(s.pool[1], s.at, x["value"].view(-1, KV_HEADS, DIM))
    return {"out": _attend(s, q, qg[:, :, 1])[0], "k": _stored(s.pool[0], s.at), "v": _stored(s.pool[1], s.at)}


# ------------------------------------------------------------------ the package's calls


def _gather(s, first, counts):
    ty = TYPES[s.case["type"]]
    s.kv.gather(LAYER, s.seqs, first, counts, s.k.data_ptr(), s.v.data_ptr(), ggml_type=ty if ty in (F16, BF16) else F32)
    return {"k": s.k, "v": s.v}


def _run_own(s):
    case = s.case
    kind, p = case["kind"], {k: v.data_ptr() for k, v in s.x.items()}
    if kind == "append":
        first, counts = [b for b, _ in s.spans], [c for _, c in s.spans]
        s.kv.append(LAYER, s.seqs, first, counts, p["k_norm"], p["key"], p["value"])
        return _gather(s, first, counts)
    zeros = [0] * len(s.seqs)
    if kind == "decode":
        s.kv.attn_decode(LAYER, s.seqs, s.positions, p["q"], s.out.data_ptr(), gate=p["gate"])
        return {"out": s.out}
    if kind == "step":
        s.kv.full_core(LAYER, s.seqs, s.positions, p["q_norm"], p["k_norm"], p["qg"], p["key"], p["value"], s.out.data_ptr())
        return dict(_gather(s, s.positions, [1] * len(s.seqs)), out=s.out)
    if kind == "evict":
        keep, recent = _kept(case)
        for q, pages in zip(s.seqs, s.lists):
            s.kv.seq_set_pages(q, pages)
        s.kv.weights_put(LAYER, s.seqs, zeros, s.counts, p["weights"])
        s.kv.evict(s.seqs, s.counts, keep, recent)
        s.kv.weights_get(LAYER, s.seqs, zeros, keep, s.weights.data_ptr(), s.tokens.data_ptr())
        return dict(_gather(s, zeros, keep), weights=s.weights, tokens=s.tokens)
    # sums of this call alone
    s.kv.weights_put(LAYER, s.seqs, zeros, s.counts)
    if kind == "observe":
        s.kv.attn_observe(LAYER, s.seqs[0], case["ctx"] - case["tokens"], case["tokens"], p["q"])
        s.kv.weights_get(LAYER, s.seqs, zeros, s.counts, s.weights.data_ptr())
        return {"weights": s.weights}
    s.kv.attn_decode(LAYER, s.seqs, s.positions, p["q"], s.out.data_ptr(), gate=p["gate"])
    s.kv.weights_get(LAYER, s.seqs, zeros, s.counts, s.weights.data_ptr())
    return {"out": s.out, "weights": s.weights}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    kind, row = case["kind"], ROW_BYTES[case["type"]]
    back = row if case["type"] in DTYPES else 4 * KV_DIM
    if kind == "append":
        n = sum(c for _, c in _pieces(case))
        return {"bytes": 2 * n * (4 * KV_DIM + 2 * row + back), "flops": 10 * n * KV_DIM}
    n, cached = len(_counts(case)), sum(_counts(case))
    if kind == "observe":
        # the keys once, the queries once, the sums once
        return {"bytes": cached * (row + 4 * KV_HEADS) + 4 * case["tokens"] * Q_DIM, "flops": 2 * case["tokens"] * cached * Q_DIM}
    if kind == "evict":
        # the weights once; the rows that stay once as they move or are handed back, and once as they are handed back
        kept = sum(_kept(case)[0])
        return {"bytes": 4 * KV_HEADS * cached + kept * (2 * row + 2 * back + 8 * KV_HEADS), "flops": cached * KV_HEADS}
    b, f = 2 * cached * row, cached * HEADS * DIM * 4
    if kind == "step":
        return {"bytes": b + 4 * n * (QG_DIM + 2 * KV_DIM + Q_DIM) + 2 * n * (row + back), "flops": f}
    return {"bytes": b + 12 * n * Q_DIM + (4 * KV_HEADS * cached if kind == "weigh" else 0), "flops": f}


# ------------------------------------------------------------------ the same in 64 bits


def _nearest4(x):
    """[n][heads][256] in 64 bits as 4-bit blocks stand for them, by the distance to each value that they can."""
    grid = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], device=x.device, dtype=torch.float64)  # even codes first: they win a tie
    out = torch.empty_like(x)
    for rows, to in zip(x.split(2048), out.split(2048)):
        b = rows.unflatten(-1, (-1, BLOCK))
        big = b.abs().amax(-1, keepdim=True)
        unit = torch.exp2(torch.ceil(torch.log2(torch.where(big == 0, 1.0, big) / 7.0)).clamp(-125, 125))
        best = (b.abs()[..., None] / unit[..., None] - grid).abs().argmin(-1)
        to.copy_((torch.sign(b) * grid[best] * unit).flatten(-2))
    return out


def _rounded(x, ty):
    """Cached rows [n][4][256] as the 64-bit numbers that their type holds."""
    if ty == "mxfp4":
        return _nearest4(x.double())
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
    kind, ty = case["kind"], case["type"]
    if kind == "append":
        # 4-bit values are a block's steps: no 64-bit value stands for them
        return None
    x, counts, at = _inputs(case, _Gen(seed)), _counts(case), 0
    if kind == "evict":
        return None if ty not in DTYPES else _evicted64(case, x)
    if kind == "observe":
        n, c = case["tokens"], case["ctx"]
        k, q = _rounded(x["k"].view(-1, KV_HEADS, DIM), ty), x["q"].double().view(n, HEADS, DIM)
        sums = torch.zeros(c, KV_HEADS, device="cuda", dtype=torch.float64)
        for h in range(HEADS):
            keys = k[:, h // GROUP].contiguous()
            for t in range(n):
                e = c - n + t + 1
                sums[:e, h // GROUP] += torch.softmax(keys[:e] @ q[t, h] / 16.0, 0)
        return {"weights": sums}
    out, sums, news = [], [], None
    if kind == "step":
        last = [c - 1 for c in counts]
        qg = x["qg"].view(-1, HEADS, 2, DIM)
        q, gate = _turned64(qg[:, :, 0], x["q_norm"], last), qg[:, :, 1].double()
        news = _turned64(x["key"].view(-1, KV_HEADS, DIM), x["k_norm"], last)
    else:
        q, gate = (x[n].double().view(-1, HEADS, DIM) for n in ("q", "gate"))
    for i, c in enumerate(counts):
        k, v = (x[n][at:at + c].view(-1, KV_HEADS, DIM) for n in ("k", "v"))
        at += c
        if news is not None:
            # the token's own rows take the last position, in the cache's type
            k = torch.cat((k[:-1], news[i:i + 1].float()))
            v = torch.cat((v[:-1], x["value"][i:i + 1].view(1, KV_HEADS, DIM)))
        k, v = _rounded(k, ty), _rounded(v, ty)
        got = torch.zeros(c, KV_HEADS, device="cuda", dtype=torch.float64)
        for h in range(HEADS):
            p = torch.softmax(k[:, h // GROUP].contiguous() @ q[i, h] / 16.0, 0)
            got[:, h // GROUP] += p
            out.append(p @ v[:, h // GROUP].contiguous() * torch.sigmoid(gate[i, h]))
        sums.append(got)
    out = torch.stack(out).view(-1, Q_DIM)
    if kind == "weigh":
        return {"out": out, "weights": torch.cat(sums)}
    return {"out": out} if news is None else {"out": out, "k": None, "v": None}


def _evicted64(case, x):
    """Head by head: whole numbers and rows as they are, with the kept positions found one at a time."""
    (keep, recent), at, parts = _kept(case), 0, []
    for c, n, r in zip(_counts(case), keep, recent):
        k, v = (x[name][at:at + c].view(-1, KV_HEADS, DIM) for name in ("k", "v"))
        w = x["weights"][at:at + c]
        at += c
        part = []
        for j in range(KV_HEADS):
            heavy = w[:, j].double().cpu().numpy().copy()
            heavy[c - r:] = np.inf
            # most weight first, then the earlier position
            stays = set(np.lexsort((np.arange(c), -heavy))[:n].tolist())
            late = iter(sorted(p for p in stays if p >= n))
            part.append([p if p in stays else next(late) for p in range(n)])
        moved = torch.tensor(part, device="cuda").t()
        heads = torch.arange(KV_HEADS, device="cuda")
        parts.append({"k": _rounded(k[moved, heads], case["type"]).reshape(n, KV_DIM),
                      "v": _rounded(v[moved, heads], case["type"]).reshape(n, KV_DIM),
                      "weights": w.gather(0, moved).double(), "tokens": moved})
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
