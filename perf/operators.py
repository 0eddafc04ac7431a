"""The decoder operators whose speed is watched: attention over a paged cache, attention of a prompt with a sliding window and
sinks, moves inside a cache, and log probabilities of tokens.

A case is a dict of plain values. `prepare` makes what a program has in hand before the call, `run` makes one call: of the
framework where `own` is set, of elementary torch operations in 32 bits otherwise. `exact` computes the same in 64 bits from the
definitions:

  paged     q[b,h] against the cached keys of its sequence and, with `new`, the key of the token itself at position p. Position
            j <= p is visible when there is no window, p - j < window, or j < sinks. A row that sees nothing is zero.
  prompt    the same for every token of a prompt; rows from a sequence's length on are zero.
  write     rows of new tokens to their slots (page * page_size + offset) of all layers' pages.
  copy      pages to other pages, keys and values of all layers.
  probs     log softmax at a row's token (0 where the token is negative), the entropy, the logarithm of the normaliser, the best
            `top` tokens (equal logits by their number); with `grad`, the gradient of the logits for given cotangents instead
            of the best tokens.

A cache is [layers, 2 (keys, values), pages, page_size, kv_heads, head_dim].
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one sequence of a chat, one shared key-value head of 256 as in the decoder of the benchmark: latency
        {"name": "paged_one", "kind": "paged", "batch": 1, "cap": 77, "heads": 8, "kv_heads": 1, "dim": 256, "page": 16,
         "window": 0, "sinks": 0, "new": True, "dtype": "bf16"},
        # a serving batch, grouped heads, sequences of every length up to 4096 in pages of 64
        {"name": "paged_batch", "kind": "paged", "batch": 32, "cap": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "window": 0, "sinks": 0, "new": True, "dtype": "f16"},
        # a 32-bit model with a head of its own for every query head, window and sinks, pages that no tile fits
        {"name": "paged_window_f32", "kind": "paged", "batch": 21, "cap": 5000, "heads": 12, "kv_heads": 12, "dim": 64, "page": 24,
         "window": 1000, "sinks": 4, "new": False, "dtype": "f32"},
        # the benchmark's prompt: 512 tokens, causal
        {"name": "prompt_512", "kind": "prompt", "batch": 1, "len": 512, "heads": 8, "kv_heads": 1, "dim": 256, "window": 0, "sinks": 0,
         "ragged": False, "dtype": "bf16"},
        # two long prompts of a model with windowed layers
        {"name": "prompt_window", "kind": "prompt", "batch": 2, "len": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "window": 1024, "sinks": 4,
         "ragged": False, "dtype": "bf16"},
        # a padded batch of a small 32-bit model, lengths that fit no tile
        {"name": "prompt_ragged_f32", "kind": "prompt", "batch": 3, "len": 501, "heads": 12, "kv_heads": 12, "dim": 64, "window": 200, "sinks": 1,
         "ragged": True, "dtype": "f32"},
        # behind a decode step of the benchmark's decoder: one row per sequence and layer
        {"name": "write_step", "kind": "write", "layers": 18, "pages": 300, "page": 16, "kv_heads": 1, "dim": 256, "rows": 16, "dtype": "bf16"},
        # behind a prompt: thousands of rows
        {"name": "write_prompt", "kind": "write", "layers": 18, "pages": 320, "page": 16, "kv_heads": 1, "dim": 256, "rows": 4099, "dtype": "bf16"},
        # copy on write: the last pages of three sequences that fork
        {"name": "copy_fork", "kind": "copy", "layers": 18, "pages": 300, "page": 16, "kv_heads": 1, "dim": 256, "pairs": 3, "dtype": "bf16"},
        # compaction: the upper half of a pool moves into holes of the lower
        {"name": "copy_compact", "kind": "copy", "layers": 6, "pages": 800, "page": 64, "kv_heads": 4, "dim": 128, "pairs": 300, "dtype": "f16"},
        # sampling and its report: a batch of vocabulary rows, the best 20 beside the token that was taken, a masked vocabulary
        {"name": "probs_serve", "kind": "probs", "rows": 8, "vocab": 256000, "top": 20, "masked": True, "grad": False, "dtype": "bf16"},
        # the loss of the masked-language-model configuration: 4096 rows of 30522 and their gradient
        {"name": "probs_train", "kind": "probs", "rows": 4096, "vocab": 30522, "top": 0, "masked": False, "grad": True, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    kind = rng.choice(["paged", "paged", "prompt", "prompt", "write", "copy", "probs", "probs"])
    kv, group, dim = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16]), rng.choice([64, 72, 96, 128, 128, 192, 256])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "paged":
        batch, page = _log(rng, 1, 64), rng.choice([1, 5, 16, 24, 32, 64, 128])
        cap = _log(rng, 1, min(131072, (1 << 26) // (batch * kv * dim), (1 << 27) // (batch * kv * group)))
        window = rng.choice([0, 0, _log(rng, 1, cap)])
        return {"kind": kind, "batch": batch, "cap": cap, "heads": kv * group, "kv_heads": kv, "dim": dim, "page": page, "window": window,
                "sinks": rng.choice([0, 1, 4, 16]) if window else 0, "new": rng.random() < 0.6, "dtype": dtype}
    if kind == "prompt":
        batch = _log(rng, 1, 8)
        most = 1 << (29 if dtype != "f32" else 27)      # scores
        n = _log(rng, 1, min(8192, int(math.sqrt(most / (batch * kv * group)))))
        window = rng.choice([0, 0, _log(rng, 1, n)])
        return {"kind": kind, "batch": batch, "len": n, "heads": kv * group, "kv_heads": kv, "dim": dim, "window": window,
                "sinks": rng.choice([0, 1, 4, 16]) if window else 0, "ragged": rng.random() < 0.5, "dtype": dtype}
    if kind in ("write", "copy"):
        layers, page, kv = _log(rng, 1, 24), rng.choice([1, 8, 16, 24, 64]), rng.choice([1, 2, 4])
        token = layers * 2 * kv * dim * SIZE[dtype]
        pages = _log(rng, 8, max(8, min(20000, (3 << 28) // (token * page))))
        case = {"kind": kind, "layers": layers, "pages": pages, "page": page, "kv_heads": kv, "dim": dim}
        case["rows" if kind == "write" else "pairs"] = _log(rng, 1, max(1, min(8192, pages * page // 2, (1 << 28) // token)) if kind == "write" else max(1, pages // 2))
        return {**case, "dtype": dtype}
    grad = rng.random() < 0.4
    vocab = _log(rng, 500, 256000)
    rows = _log(rng, 1, max(1, min(8192, 125_000_000 // vocab)) if grad else max(1, min(2048, 60_000_000 // vocab)))
    return {"kind": kind, "rows": rows, "vocab": vocab, "top": 0 if grad else rng.choice([0, 1, 5, 20, 64]), "masked": rng.random() < 0.5,
            "grad": grad, "dtype": dtype}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _lengths(c):
    """Tokens of each sequence, in some order: spread evenly over the range, a padding row of none in a batch of four and more."""
    B, cap = c["batch"], c["cap"]
    if B < 4:
        return [cap * (i + 1) // B for i in range(B)]
    return [cap * i // (B - 1) for i in range(B)]


def _prompt_lengths(c):
    B, n = c["batch"], c["len"]
    return [n - (2 * n // 3) * i // max(1, B - 1) for i in range(B)] if c["ragged"] else [n] * B


def _inputs(c, seed):
    """The arguments of a case by name: tensors on the device, and for the moves inside a cache numpy arrays of indices."""
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    host = np.random.default_rng(seed)

    def normal(*shape, std=1.0, dtype=c["dtype"]):
        return torch.empty(shape, dtype=TORCH[dtype], device=dev).normal_(0.0, std, generator=g)

    def ints(values):
        return torch.tensor(np.asarray(values, np.int32), device=dev)

    kind = c["kind"]
    if kind == "paged":
        lens = host.permutation(np.asarray(_lengths(c), np.int32))
        per = [-(-int(n) // c["page"]) for n in lens]
        width = -(-c["cap"] // c["page"])
        pages = sum(per) + 3
        order, table, at = host.permutation(pages), np.full((c["batch"], width), -1, np.int32), 0
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        d = {"q": normal(c["batch"], c["heads"], c["dim"]), "cache": normal(1, 2, pages, c["page"], c["kv_heads"], c["dim"]),
             "table": ints(table), "lengths": ints(lens)}
        if c["new"]:
            d["new"] = normal(2, c["batch"], c["kv_heads"], c["dim"])
        return d
    if kind == "prompt":
        B, T = c["batch"], c["len"]
        return {"q": normal(B, T, c["heads"], c["dim"]), "k": normal(B, T, c["kv_heads"], c["dim"]), "v": normal(B, T, c["kv_heads"], c["dim"]),
                "lengths": ints(host.permutation(np.asarray(_prompt_lengths(c))))}
    if kind in ("write", "copy"):
        d = {"cache": normal(c["layers"], 2, c["pages"], c["page"], c["kv_heads"], c["dim"])}
        if kind == "write":
            d["rows"] = normal(c["layers"], 2, c["rows"], c["kv_heads"], c["dim"])
            d["slots"] = host.permutation(c["pages"] * c["page"])[:c["rows"]].astype(np.int32)
        else:
            order = host.permutation(c["pages"])
            d["pairs"] = np.stack([order[:c["pairs"]], order[::-1][:c["pairs"]]], 1).astype(np.int32)
        return d
    R, V = c["rows"], c["vocab"]
    x = normal(R, V, std=3.0)
    if c["masked"]:
        x.masked_fill_(torch.rand((V,), generator=g, device=dev) < 0.3, -math.inf)
    tokens = host.integers(0, V, R)
    if c["masked"]:                                      # the tokens that were taken are among those that were allowed
        free = torch.nonzero(torch.isfinite(x[0])).flatten().cpu().numpy()
        tokens = free[tokens % len(free)]
    if c["grad"]:
        tokens[::7] = -1                                 # rows without a label
    d = {"logits": x, "tokens": ints(tokens)}
    if c["grad"]:
        d["d_log_prob"], d["d_entropy"], d["d_normalizer"] = (normal(R, std=s, dtype="f32") for s in (1.0 / R, 0.01 / R, 0.01 / R))
    return d


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
_client = None
_executables = {}
_stage = None


def _framework():
    global _client
    sys.path.insert(0, os.path.join(os.getcwd(), "jax-mps_b200"))
    import b200
    if _client is None:
        _client = b200.Client(device_ordinal=0)
    return _client


def _put(t):
    """A device tensor as a buffer of the client, through pinned host memory."""
    global _stage
    size = t.numel() * t.element_size()
    if _stage is None or _stage.numel() < size:
        _stage = torch.empty(max(size, 64 << 20), dtype=torch.uint8, pin_memory=True)
    host = _stage[:size].view(t.dtype).view(t.shape)
    host.copy_(t)
    if t.dtype == torch.bfloat16:
        buf = _client.buffer_from_host(host.view(torch.int16).numpy().view(np.uint16), dtype="bf16")
    else:
        buf = _client.buffer_from_host(host.numpy())
    _client.synchronize()              # the staging memory is free again
    return buf


def _program(c, args):
    """The program of one operator: its module text and the types of its results."""
    from b200.shlo.builder import Builder
    names = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16", torch.int32: "i32"}
    b = Builder()
    a = {n: b.arg(tuple(t.shape), names[t.dtype]) for n, t in args.items()}
    if c["kind"] == "paged":
        outs = [b.paged_attention(a["q"], a["cache"], a["table"], a["lengths"], new=a.get("new"), window=c["window"], sinks=c["sinks"])]
    elif c["kind"] == "prompt":
        outs = [b.window_attention(a["q"], a["k"], a["v"], a["lengths"], window=c["window"], sinks=c["sinks"])]
    else:
        outs = b.token_log_probs(a["logits"], a["tokens"], top=c["top"])
        if c["grad"]:
            terms = [b.mul(y, a[d]) for y, d in zip(outs, ("d_log_prob", "d_entropy", "d_normalizer"))]
            outs += b.grad(b.reduce_sum(b.add(b.add(terms[0], terms[1]), terms[2]), (0,)), [a["logits"]])
    return b.module(outs), [(o.shape, o.dtype) for o in outs]


class Outputs(list):
    """The result buffers of one call. A user's program hands them to its next call as they are; here each becomes a tensor when
    it is read."""

    def __init__(self, bufs, types):
        super().__init__(bufs)
        self.types = types

    def __iter__(self):
        _client.synchronize()
        for buf, (shape, dtype) in zip(super().__iter__(), self.types):
            t = torch.as_tensor(_View(buf, shape, dtype), device="cuda")
            yield t.view(torch.bfloat16) if dtype == "bf16" else t


class _View:
    def __init__(self, buf, shape, dtype):
        self.buf = buf
        self.__cuda_array_interface__ = {"data": (buf.device_pointer(), False), "shape": tuple(shape), "version": 3,
                                         "typestr": {"f32": "<f4", "f16": "<f2", "bf16": "<i2", "i32": "<i4"}[dtype]}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.case = case
    args = _inputs(case, seed)
    if own:
        client = _framework()
        if case["kind"] in ("write", "copy"):
            s.exe, s.types = client, [(args["cache"].shape, case["dtype"])]
            s.args = {n: t if isinstance(t, np.ndarray) else _put(t) for n, t in args.items()}
            return s
        key = tuple(sorted((k, v) for k, v in case.items() if k != "name"))
        # the widths of tables and caches follow from the case alone
        if key not in _executables:
            text, types = _program(case, args)
            _executables[key] = (client.compile(text), types)
        s.exe, s.types = _executables[key]
        s.args = [_put(t) for t in args.values()]
        return s
    s.args = {n: torch.from_numpy(t).cuda().long() if isinstance(t, np.ndarray) else t for n, t in args.items()}
    return s


def run(state):
    c, a = state.case, state.args
    if own:
        if c["kind"] == "write":
            state.exe.write_pages(a["cache"], a["rows"], a["slots"])
            return Outputs([a["cache"]], state.types)
        if c["kind"] == "copy":
            state.exe.copy_pages(a["cache"], a["pairs"])
            return Outputs([a["cache"]], state.types)
        return Outputs(state.exe.execute(a), state.types)
    return {"paged": _paged, "prompt": _prompt, "write": _write, "copy": _copy, "probs": _probs}[c["kind"]](c, **a)


def _visible(c, p, j):
    """Whether position j is among those that a query at position p sees."""
    see = j <= p
    return see & ((p - j < c["window"]) | (j < c["sinks"])) if c["window"] else see


def _softmax(s, see):
    s = torch.where(see, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.where(see, torch.exp(s - torch.where(m == -math.inf, 0.0, m)), 0.0)
    return e / e.sum(-1, keepdim=True).clamp_min(1e-37)


def _paged(c, q, cache, table, lengths, new=None):
    B, KH, D, G = c["batch"], c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"]
    k, v = (cache[0, i][table.clamp_min(0)].flatten(1, 2).float() for i in (0, 1))          # [B, positions, KH, D]
    j = torch.arange(k.shape[1], device=q.device).expand(B, -1)
    there, p = j < lengths[:, None], lengths[:, None] - 1
    if new is not None:
        k, v = (torch.cat([t, new[i][:, None].float()], 1) for i, t in enumerate((k, v)))
        p = p + 1
        j, there = torch.cat([j, p], 1), torch.cat([there, torch.ones_like(there[:, :1])], 1)
    see = (there & _visible(c, p, j))[:, None, None]
    s = torch.einsum("bhgd,bthd->bhgt", q.view(B, KH, G, D).float(), k) * D ** -0.5
    o = torch.einsum("bhgt,bthd->bhgd", _softmax(s, see), v)
    return [o.reshape(q.shape).to(q.dtype)]


def _prompt(c, q, k, v, lengths):
    B, T, KH, D = k.shape
    at = torch.arange(T, device=q.device)
    see = _visible(c, at[:, None], at) & (at[:, None] < lengths[:, None, None])                # [B, T, T]
    s = torch.einsum("bqhgd,bkhd->bhgqk", q.view(B, T, KH, -1, D).float(), k.float()) * D ** -0.5
    o = torch.einsum("bhgqk,bkhd->bqhgd", _softmax(s, see[:, None, None]), v.float())
    return [o.reshape(q.shape).to(q.dtype)]


def _write(c, cache, rows, slots):
    cache.flatten(2, 3)[:, :, slots] = rows
    return [cache]


def _copy(c, cache, pairs):
    cache[:, :, pairs[:, 1]] = cache[:, :, pairs[:, 0]]
    return [cache]


def _probs(c, logits, tokens, d_log_prob=None, d_entropy=None, d_normalizer=None):
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    norm = m + torch.log(total)
    entropy = torch.log(total) - torch.where(e > 0, e * (x - m), 0.0).sum(-1, keepdim=True) / total
    known = (tokens >= 0)[:, None]
    at = tokens.clamp_min(0).long()[:, None]
    lp = torch.where(known, x.gather(1, at) - norm, 0.0)
    outs = [lp[:, 0], entropy[:, 0], norm[:, 0]]
    if c["top"]:
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)                               # floats in order as integers
        key = (order << 32) + (c["vocab"] - 1 - torch.arange(c["vocab"], device=x.device))   # equal ones by their number
        ids = key.topk(c["top"], -1).indices
        outs += [x.gather(1, ids) - norm, ids.int()]
    if c["grad"]:
        p = e / total
        dlp, dh, dn = (t[:, None] for t in (d_log_prob, d_entropy, d_normalizer))
        dlp = torch.where(known, dlp, 0.0)
        dx = p * (dn - dlp) - dh * torch.where(p > 0, p * (x - norm + entropy), 0.0)
        outs.append(dx.scatter_add(1, at, dlp).to(logits.dtype))
    return outs


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _attend(q, k, v):
    """One query row after another would be the definition; here all query heads [G, D] of one key-value head and one position."""
    if k.shape[0] == 0:
        return torch.zeros_like(q)
    s = q @ k.T / math.sqrt(q.shape[-1])
    w = (s - s.logsumexp(-1, keepdim=True)).exp()
    return w @ v


def exact(case, seed):
    c, a = case, _inputs(case, seed)
    kind = c["kind"]
    if kind == "paged":
        q, cache = a["q"].double(), a["cache"][0]
        out = torch.zeros_like(q)
        G = c["heads"] // c["kv_heads"]
        for b in range(c["batch"]):
            n = int(a["lengths"][b])
            p = n if c["new"] else n - 1
            js = [j for j in range(n) if not c["window"] or p - j < c["window"] or j < c["sinks"]]
            slots = torch.tensor([int(x) for x in js], device=q.device, dtype=torch.long)
            slots = a["table"][b].long()[slots // c["page"]] * c["page"] + slots % c["page"]
            kv = cache.flatten(1, 2)[:, slots].double()                                      # [2, n, KH, D]
            if c["new"]:
                kv = torch.cat([kv, a["new"][:, b:b + 1].double()], 1)
            for h in range(c["kv_heads"]):
                out[b, h * G:(h + 1) * G] = _attend(q[b, h * G:(h + 1) * G], kv[0, :, h], kv[1, :, h])
        return [out]
    if kind == "prompt":
        out = torch.zeros(a["q"].shape, dtype=torch.float64, device=a["q"].device)
        G = c["heads"] // c["kv_heads"]
        for b in range(c["batch"]):
            n = int(a["lengths"][b])
            i = torch.arange(n, device=out.device)
            gap = i[:, None] - i[None]
            hidden = gap < 0
            if c["window"]:
                hidden |= (gap >= c["window"]) & (i >= c["sinks"])
            for h in range(c["heads"]):
                s = a["q"][b, :n, h].double() @ a["k"][b, :n, h // G].double().T / math.sqrt(c["dim"])
                s.masked_fill_(hidden, -math.inf)
                out[b, :n, h] = (s - s.logsumexp(-1, keepdim=True)).exp() @ a["v"][b, :n, h // G].double()
        return [out]
    if kind == "write":
        flat = a["cache"].flatten(2, 3)
        for r, slot in enumerate(a["slots"].tolist()):
            flat[:, :, slot] = a["rows"][:, :, r]
        return [a["cache"]]
    if kind == "copy":
        old = a["cache"].clone()
        for src, dst in a["pairs"].tolist():
            a["cache"][:, :, dst] = old[:, :, src]
        return [a["cache"]]
    parts, step = [], max(1, 20_000_000 // c["vocab"])
    for r in range(0, c["rows"], step):
        x = a["logits"][r:r + step].double()
        t = a["tokens"][r:r + step].long()
        logp = x - x.logsumexp(-1, keepdim=True)
        p = logp.exp()
        h = -torch.where(p > 0, p * logp, 0.0).sum(-1)
        hot = torch.zeros_like(x)
        hot[torch.arange(len(t), device=x.device)[t >= 0], t[t >= 0]] = 1.0
        row = [torch.where(hot > 0, logp, 0.0).sum(-1), h, x.logsumexp(-1)]
        if c["top"]:
            best = torch.sort(x, dim=-1, descending=True, stable=True)
            row += [best.values[:, :c["top"]] - row[2][:, None], best.indices[:, :c["top"]].int()]
        if c["grad"]:
            dl, dh, dn = (a[n][r:r + step].double()[:, None] for n in ("d_log_prob", "d_entropy", "d_normalizer"))
            dx = dl * torch.where((t >= 0)[:, None], hot - p, 0.0) + dn * p
            row.append(dx - dh * torch.where(p > 0, p * (logp + h[:, None]), 0.0))
        parts.append(row)
    return [torch.cat(col) for col in zip(*parts)]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c, kind, size = case, case["kind"], SIZE[case["dtype"]]
    if kind == "paged":
        seen = 0
        for n in _lengths(c):
            first = max(0, (n if c["new"] else n - 1) - c["window"] + 1) if c["window"] else 0
            seen += min(n, n - first + min(c["sinks"], first))
        rows = seen + (c["batch"] if c["new"] else 0)
        pages = -(-seen // c["page"])
        return {"bytes": size * (2.0 * rows * c["kv_heads"] * c["dim"] + 2.0 * c["batch"] * c["heads"] * c["dim"]) + 4.0 * (pages + c["batch"]),
                "flops": 4.0 * rows * c["heads"] * c["dim"]}
    if kind == "prompt":
        pairs = 0
        for n in _prompt_lengths(c):
            w = min(c["window"] or n, n)
            pairs += w * (w + 1) // 2 + (n - w) * w
            far = n - w                                        # rows with positions behind their window
            s = min(c["sinks"], far)
            pairs += s * (s + 1) // 2 + (far - s) * s          # a row sees one more of the sinks for each step past the window
        rows = sum(_prompt_lengths(c))
        return {"bytes": size * c["dim"] * (rows * (c["heads"] + 2.0 * c["kv_heads"]) + c["batch"] * c["len"] * c["heads"]),
                "flops": 4.0 * pairs * c["heads"] * c["dim"]}
    if kind in ("write", "copy"):
        token = c["layers"] * 2 * c["kv_heads"] * c["dim"] * size
        moved = c["rows"] if kind == "write" else c["pairs"] * c["page"]
        return {"bytes": 2.0 * moved * token, "flops": 0.0}
    R, V = c["rows"], c["vocab"]
    return {"bytes": R * V * size * (2.0 if c["grad"] else 1.0) + R * (16.0 + 8 * c["top"] + (12 if c["grad"] else 0)), "flops": 5.0 * R * V}
