"""The serving operators, measured one pass at a time: keys and values rotated
into a paged cache, attention over that cache and over plain tensors with a
sliding window and a few first tokens that stay visible, and the draw of the
next token.

A paged cache is two arrays (pages, page, kv_heads, dim); a sequence's row of
``block_tables`` names its pages in order (-1: none), ``context_lens`` counts
its tokens, the new ones included, and ``query_starts`` (sequences + 1) says
where its new tokens begin in the packed batch (left out where every sequence
has one).  The query at position p sees key j where j <= p and
p - j < window or j < sinks.

Case kinds and what they vary:

  append   tokens, seqs, context, heads, kv_heads, dim, rotary, page, dtype
  paged    tokens, seqs, context, heads, kv_heads, dim, page, window, sinks, dtype
  window   batch, seq, heads, kv_heads, dim, window, sinks, padded, dtype
  sample   rows, vocab, top_k, top_p, min_p, dtype

``tokens`` 0 is one new token for each sequence, ``window`` 0 is none.
"""

import math
import random

import numpy as np
import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NAME = {torch.bfloat16: "bfloat16", torch.float16: "float16", torch.float32: "float32", torch.int32: "int32"}
ROPE_BASE = 1.0e6


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    heads = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16"}
    return [
        # One decode step of a few sequences: the call's own latency.
        {"name": "append_step", "kind": "append", "tokens": 0, "seqs": 8, "context": 4000, "rotary": 128, **heads},
        # A batch of prompts, some with a cached beginning, of lengths nobody
        # rounded.
        {"name": "append_prompts", "kind": "append", "tokens": 8000, "seqs": 6, "context": 5000, "rotary": 128, **heads},
        # One sequence generating.
        {"name": "paged_one", "kind": "paged", "tokens": 0, "seqs": 1, "context": 1500, "window": 0, "sinks": 0, **heads},
        # A full batch generating, contexts of many lengths.
        {"name": "paged_batch", "kind": "paged", "tokens": 0, "seqs": 64, "context": 8192, "window": 0, "sinks": 0,
         **heads},
        # Long conversations of a model with a sliding window: a few sequences,
        # of which a window and the first tokens are read.
        {"name": "paged_window", "kind": "paged", "tokens": 0, "seqs": 16, "context": 60000, "window": 4096, "sinks": 4,
         **heads, "page": 32, "dtype": "f16"},
        # A scheduler's step: chunks of prompts next to generating sequences.
        {"name": "paged_chunks", "kind": "paged", "tokens": 2100, "seqs": 24, "context": 6000, "window": 1024,
         "sinks": 4, **heads},
        # Two short prompts.
        {"name": "window_short", "kind": "window", "batch": 2, "seq": 333, "heads": 16, "kv_heads": 8, "dim": 128,
         "window": 128, "sinks": 4, "padded": True, "dtype": "bf16"},
        # A small model with as many key heads as query heads.
        {"name": "window_dim64", "kind": "window", "batch": 4, "seq": 2000, "heads": 16, "kv_heads": 16, "dim": 64,
         "window": 512, "sinks": 1, "padded": False, "dtype": "f16"},
        # A long prompt (the largest case).
        {"name": "window_long", "kind": "window", "batch": 1, "seq": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 4096, "sinks": 16, "padded": False, "dtype": "bf16"},
        # The token of one sequence, a small vocabulary.
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 32000, "top_k": 50, "top_p": 0.9, "min_p": 0.0,
         "dtype": "f32"},
        # A batch's tokens over a large vocabulary, every filter on.
        {"name": "sample_batch", "kind": "sample", "rows": 64, "vocab": 151936, "top_k": 200, "top_p": 0.95,
         "min_p": 0.02, "dtype": "bf16"},
        # The nucleus alone, of a vocabulary in odd pieces.
        {"name": "sample_nucleus", "kind": "sample", "rows": 17, "vocab": 128257, "top_k": 0, "top_p": 0.9, "min_p": 0.0,
         "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    """An integer from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


_HEADS = [(32, 8, 128), (16, 8, 128), (16, 2, 128), (8, 8, 128), (40, 8, 128), (16, 16, 64), (24, 8, 64), (32, 1, 64)]
_PAGES = [16, 16, 32, 64, 24, 128]
MOST_FLOPS = 5e11
MOST_BYTES = 2e9


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES:
            return c


def _draw(rng):
    kind = rng.choice(["append", "paged", "paged", "window", "window", "sample", "sample"])
    c = {"kind": kind}
    if kind == "sample":
        c.update(rows=_log(rng, 1, 256), vocab=_log(rng, 500, 260000), top_k=rng.choice([0, 0, 1, 20, _log(rng, 2, 5000)]),
                 top_p=rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]),
                 dtype=rng.choice(["bf16", "f32", "f16"]))
        return c
    heads, kv, dim = rng.choice(_HEADS)
    c.update(heads=heads, kv_heads=kv, dim=dim, dtype=rng.choice(["bf16", "bf16", "f16"]))
    if kind == "window":
        seq = _log(rng, 1, 8192)
        c.update(batch=_log(rng, 1, max(1, min(32, 16384 // seq))), seq=seq, window=rng.choice([0, _log(rng, 1, 4096)]),
                 padded=rng.random() < 0.5)
    else:
        seqs = _log(rng, 1, 128)
        c.update(seqs=seqs, context=_log(rng, 16, min(65536, 262144 // seqs)), page=rng.choice(_PAGES),
                 tokens=rng.choice([0, seqs + _log(rng, 1, 4096)]))
        if kind == "append":
            c["rotary"] = rng.choice([dim, dim, dim // 2])
            return c
        c["window"] = rng.choice([0, _log(rng, 16, 8192)])
    c["sinks"] = rng.choice([0, 1, 4, 40]) if c["window"] else 0
    return c


def _sequences(c):
    """(new tokens, context lengths) of each sequence, from the case alone."""
    r = random.Random("%d %d %d" % (c["seqs"], c["context"], c["tokens"]))
    n = c["seqs"]
    new = [1] * n
    if c["tokens"]:  # two in three sequences share what is left of the tokens
        share = [r.random() if b == 0 or r.random() < 0.67 else 0.0 for b in range(n)]
        left = c["tokens"] - n
        for b in range(n):
            new[b] += int(left * share[b] / sum(share))
        new[0] += c["tokens"] - sum(new)
    lens = [max(new[b], c["context"] if b == 0 else int(c["context"] * r.uniform(0.05, 1.0)), 1) for b in range(n)]
    return new, lens


# ---------------------------------------------------------------------------
# What a program has in hand before the call
# ---------------------------------------------------------------------------
def _inputs(c, seed):
    """Named inputs of the case on the GPU, in the kernels' argument order."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype = TORCH[c["dtype"]]

    def normal(shape, std=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if c["kind"] == "sample":
        rows, vocab = c["rows"], c["vocab"]
        x = torch.randn((rows, vocab), generator=gen, device="cuda") * 2.0
        # a trained model's logits have a few leaders in each row
        lead = torch.randint(0, vocab, (rows, 12), generator=gen, device="cuda")
        x.scatter_add_(1, lead, torch.rand((rows, 12), generator=gen, device="cuda") * 14.0)
        return {"logits": x.to(dtype), "uniform": torch.rand(rows, generator=gen, device="cuda"),
                "temperature": 0.5 + torch.rand(rows, generator=gen, device="cuda")}
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "window":
        b, s = c["batch"], c["seq"]
        d = {"qkv": normal((b, s, heads + 2 * kv, dim))}
        if c["padded"]:
            r = random.Random("%d %d" % (b, s))
            d["lengths"] = ints([s if i == 0 else r.randint(max(1, s // 4), s) for i in range(b)])
        return d
    new, lens = _sequences(c)
    n, page = sum(new), c["page"]
    need = [-(-x // page) for x in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").cpu().tolist()
    table, at = [], 0
    for k in need:
        table.append(order[at:at + k] + [-1] * (max(need) - k))
        at += k
    d = {}
    if c["kind"] == "append":
        half, most = c["rotary"] // 2, max(lens)
        angle = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * ROPE_BASE ** (
            -torch.arange(half, dtype=torch.float64, device="cuda") / half)
        d.update(qkv=normal((n, heads + 2 * kv, dim)), cos=angle.cos().float(), sin=angle.sin().float())
    else:
        d["q"] = normal((n, heads, dim))
    d.update(key_cache=normal((pages, page, kv, dim)), value_cache=normal((pages, page, kv, dim)),
             block_tables=ints(table), context_lens=ints(lens))
    if c["tokens"]:
        d["query_starts"] = ints(np.cumsum([0] + new).tolist())
    return d


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _load(case, t)
    t["case"] = dict(case)
    if case["kind"] in ("append", "paged"):  # the lengths, as the program that batched the sequences knows them
        t["new"], t["lens"] = _sequences(case)
    elif case["kind"] == "window":
        t["lens"] = t["lengths"].tolist() if case["padded"] else [case["seq"]] * case["batch"]
    return t


# ---------------------------------------------------------------------------
# The framework's operators
# ---------------------------------------------------------------------------
def _kernels():
    from nkipy_amd.core import tensor_apis

    def append(qkv, cos, sin, key_cache, value_cache, block_tables, context_lens, query_starts, heads, kv_heads):
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        return tensor_apis.rotary_append(q, k, v, cos, sin, key_cache, value_cache, block_tables, context_lens,
                                         query_starts)

    def paged(q, key_cache, value_cache, block_tables, context_lens, query_starts, window, sinks):
        return tensor_apis.paged_attention(q, key_cache, value_cache, block_tables, context_lens, query_starts,
                                           window=window, sinks=sinks)

    def window(qkv, lengths, heads, kv_heads, window, sinks):
        q, k, v = qkv[:, :, :heads], qkv[:, :, heads:heads + kv_heads], qkv[:, :, heads + kv_heads:]
        return tensor_apis.window_attention(q, k, v, lengths, window=window, sinks=sinks)

    def sample(logits, uniform, temperature, top_k, top_p, min_p):
        return tensor_apis.sample(logits, uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)

    return {"append": append, "paged": paged, "window": window, "sample": sample}


class _Memory:
    """A DeviceTensor's buffer as torch sees it (no copy); a torch view keeps
    this object, and with it the buffer, alive."""

    _TYPES = {2: "<i2", 4: "<i4"}

    def __init__(self, t, itemsize):
        self.owner = t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": self._TYPES[itemsize], "data": (t.ptr, False),
                                         "version": 2}


def _load(c, t):
    from nkipy_amd.runtime import DeviceKernel, DeviceTensor

    view = lambda x, d: torch.as_tensor(_Memory(x, d.itemsize), device="cuda").view(d)  # noqa: E731
    dev = {}
    for n in list(t):
        x = t.pop(n)
        dev[n] = DeviceTensor.empty(tuple(x.shape), NAME[x.dtype], name=n)
        view(dev[n], x.dtype).copy_(x)
        del x
    kind = c["kind"]
    if kind == "append":
        rest = dict(query_starts=dev.get("query_starts"), heads=c["heads"], kv_heads=c["kv_heads"])
    elif kind == "paged":
        rest = dict(query_starts=dev.get("query_starts"), window=c["window"] or None, sinks=c["sinks"])
    elif kind == "window":
        rest = dict(lengths=dev.get("lengths"), heads=c["heads"], kv_heads=c["kv_heads"], window=c["window"] or None,
                    sinks=c["sinks"])
    else:
        rest = dict(top_k=c["top_k"] or None, top_p=c["top_p"] if c["top_p"] < 1 else None, min_p=c["min_p"] or None)
    dk = DeviceKernel.compile_and_load(_kernels()[kind], name="perf_" + kind, **{**dev, **rest})
    alias = ".must_alias_input"
    inputs = {n: dev[n.split(alias)[0]] for n in dk.input_tensors_info}
    outputs, views = {}, {}
    for n, info in dk.output_tensors_info.items():
        outputs[n] = dev[n] if n in dev else DeviceTensor.empty(tuple(info.shape), info.dtype, name=n)
        views[n] = view(outputs[n], getattr(torch, info.dtype))
    torch.cuda.synchronize()
    return {"kernel": dk, "inputs": inputs, "outputs": outputs, "views": views}


def run(state):
    if own:
        # steps of a serving loop queue
        state["kernel"](state["inputs"], state["outputs"], sync=False)
        return state["views"]
    return _PLAIN[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _rows(s, b, upto):
    """Flat cache rows of the positions 0 .. upto-1 of sequence b."""
    page = s["case"]["page"]
    at = torch.arange(upto, device="cuda")
    return s["block_tables"][b].long()[at // page] * page + at % page


def _plain_append(s):
    c = s["case"]
    heads, kv, dim, half = c["heads"], c["kv_heads"], c["dim"], c["rotary"] // 2
    if "query_starts" in s:
        new = (s["query_starts"][1:] - s["query_starts"][:-1]).long()
        starts = s["query_starts"][:-1].long()
        seq = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), new, output_size=s["qkv"].shape[0])
        pos = s["context_lens"].long()[seq] - new[seq] + torch.arange(seq.numel(), device="cuda") - starts[seq]
    else:
        seq = torch.arange(c["seqs"], device="cuda")
        pos = s["context_lens"].long() - 1
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    x = s["qkv"][:, :heads + kv].float()
    x0, x1 = x[..., :half], x[..., half:2 * half]
    x = torch.cat([x0 * cos - x1 * sin, x0 * sin + x1 * cos, x[..., 2 * half:]], -1).to(s["qkv"].dtype)
    row = s["block_tables"].long()[seq, pos // c["page"]] * c["page"] + pos % c["page"]
    s["key_cache"].view(-1, kv, dim)[row] = x[:, heads:]
    s["value_cache"].view(-1, kv, dim)[row] = s["qkv"][:, heads + kv:]
    return {"output0": x[:, :heads].contiguous(), "key_cache": s["key_cache"], "value_cache": s["value_cache"]}


def _plain_rows(q, k, v, first, window, sinks):
    """Attention of the queries q (n, heads, dim), at positions first ..., to
    the keys and values k, v (length, kv, dim), a piece of the queries at a
    time, in 32 bits."""
    n, heads, dim = q.shape
    kv = k.shape[1]
    rep = heads // kv
    out = torch.zeros((n, heads, dim), dtype=torch.float32, device=q.device)
    step = 512
    for a in range(0, n, step):
        m = min(step, n - a)
        lo, hi = first + a, min(first + a + m, k.shape[0])
        if hi <= 0:
            continue
        low = max(0, lo - window + 1) if window else 0
        kk, vv = k[low:hi], v[low:hi]
        j = torch.arange(low, hi, device=q.device)
        if min(sinks, low):
            kk, vv = torch.cat([k[:min(sinks, low)], kk]), torch.cat([v[:min(sinks, low)], vv])
            j = torch.cat([torch.arange(min(sinks, low), device=q.device), j])
        p = torch.arange(lo, lo + m, device=q.device)[:, None]
        seen = j <= p
        if window:
            seen = seen & ((p - j < window) | (j < sinks))
        x = q[a:a + m].float().reshape(m, kv, rep, dim).permute(1, 2, 0, 3).reshape(kv, rep * m, dim)
        x = torch.bmm(x, kk.float().permute(1, 2, 0).contiguous()).reshape(kv, rep, m, -1) * (1.0 / math.sqrt(dim))
        x = x.masked_fill(~seen, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        total = x.sum(-1, keepdim=True)
        o = torch.bmm(x.reshape(kv, rep * m, -1), vv.float().permute(1, 0, 2).contiguous()).reshape(kv, rep, m, dim)
        out[a:a + m] = (o / total).permute(2, 0, 1, 3).reshape(m, heads, dim)
    return out.to(q.dtype)


def _plain_paged(s):
    c, at, parts = s["case"], 0, []
    for b in range(c["seqs"]):
        row = _rows(s, b, s["lens"][b])
        k, v = (s[x].view(-1, c["kv_heads"], c["dim"])[row] for x in ("key_cache", "value_cache"))
        n = s["new"][b]
        parts.append(_plain_rows(s["q"][at:at + n], k, v, s["lens"][b] - n, c["window"], c["sinks"]))
        at += n
    return {"output0": torch.cat(parts)}


def _plain_window(s):
    c = s["case"]
    heads, kv = c["heads"], c["kv_heads"]
    out = torch.zeros((c["batch"], c["seq"], heads, c["dim"]), dtype=s["qkv"].dtype, device="cuda")
    for b in range(c["batch"]):
        x = s["qkv"][b, :s["lens"][b]]
        out[b, :s["lens"][b]] = _plain_rows(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], 0, c["window"],
                                            c["sinks"])
    return {"output0": out}


def _plain_sample(s):
    c = s["case"]
    x = s["logits"].double()  # the draw is a comparison of long sums
    x = (x - x.amax(-1, keepdim=True)) / s["temperature"].double()[:, None]
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp(x)
    keep = torch.ones_like(w, dtype=torch.bool)
    if c["top_k"]:
        keep[:, c["top_k"]:] = False
    if c["top_p"] < 1:
        total = torch.cumsum(w * keep, -1)
        keep &= (total - w * keep) < c["top_p"] * total[:, -1:]
    if c["min_p"]:
        keep &= w >= c["min_p"]
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order, w * keep)  # in the order of the vocabulary
    total = torch.cumsum(w, -1)
    return {"output0": (total <= s["uniform"].double()[:, None] * total[:, -1:]).sum(-1).to(torch.int32)}


_PLAIN = {"append": _plain_append, "paged": _plain_paged, "window": _plain_window, "sample": _plain_sample}


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------
def _pairs(n, first, length, window, sinks):
    """(visible pairs, keys seen by any) of n queries at positions first ..."""
    pairs, last = 0, min(first + n, length)
    for p in range(first, last):
        low = max(0, p - window + 1) if window else 0
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, first - window + 1) if window else 0
    return pairs, max(0, last - low) + min(sinks, low)


def work(case):
    c = case
    size = {"bf16": 2, "f16": 2, "f32": 4}[c["dtype"]]
    if c["kind"] == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * size + 12), "flops": 3 * c["rows"] * c["vocab"]}
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "window":
        r = random.Random("%d %d" % (c["batch"], c["seq"]))
        s = c["seq"]
        lens = [s if i == 0 or not c["padded"] else r.randint(max(1, s // 4), s) for i in range(c["batch"])]
        pairs = sum(_pairs(n, 0, n, c["window"], c["sinks"])[0] for n in lens)
        return {"bytes": (sum(lens) * (heads + 2 * kv) + c["batch"] * s * heads) * dim * size,
                "flops": 4 * pairs * heads * dim}
    new, lens = _sequences(c)
    n = sum(new)
    if c["kind"] == "append":
        return {"bytes": 2 * n * (heads + 2 * kv) * dim * size + 4 * n * c["rotary"], "flops": 3 * n * (heads + kv) * c["rotary"]}
    seen = [_pairs(a, b - a, b, c["window"], c["sinks"]) for a, b in zip(new, lens)]
    return {"bytes": (2 * n * heads + 2 * sum(k for _, k in seen) * kv) * dim * size,
            "flops": 4 * sum(p for p, _ in seen) * heads * dim}


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------
def _head64(q, k, v, seen):
    """One head: q (n, dim), k, v (m, dim), seen (n, m)."""
    s = (q @ k.t().contiguous()) * q.shape[1] ** -0.5
    s = torch.softmax(torch.where(seen, s, torch.full_like(s, -math.inf)), -1)
    return s @ v


def _attend64(q, k, v, first, window, sinks):
    n, heads, dim = q.shape
    rep, out = heads // k.shape[1], torch.zeros((n, heads, dim), dtype=torch.float64, device=q.device)
    for a in range(0, n, 2048):
        z = min(n, a + 2048)
        pos = first + torch.arange(a, z, device=q.device).unsqueeze(1)
        key = torch.arange(min(k.shape[0], first + z), device=q.device)
        if window:  # the keys that any of these queries sees
            key = key[(key < sinks) | (key > first + a - window)]
        hidden = (key > pos) | ((key <= pos - window) & (key >= sinks) if window else torch.zeros_like(key, dtype=torch.bool))
        for g in range(k.shape[1]):
            kk, vv = k[key, g].double(), v[key, g].double()
            for h in range(g * rep, g * rep + rep):
                out[a:z, h] = _head64(q[a:z, h].double(), kk, vv, ~hidden)
    return out


def _sample64(c, t):
    """Row by row on the host: the definition, in float64."""
    logits, u, temp = t["logits"].double().cpu().numpy(), t["uniform"].double().cpu().numpy(), t["temperature"].double().cpu().numpy()
    ids = np.zeros(c["rows"], np.int32)
    for r in range(c["rows"]):
        z = logits[r] / temp[r]
        order = np.argsort(-z, kind="stable")
        p = np.exp(z[order] - z[order[0]])
        n = min(c["top_k"] or c["vocab"], c["vocab"])
        if c["top_p"] < 1:
            mass = np.cumsum(p[:n])
            n = min(n, 1 + int(np.searchsorted(mass, c["top_p"] * mass[-1], side="left")))
        if c["min_p"]:
            n = min(n, int(np.count_nonzero(p[:n] >= c["min_p"])))
        kept = np.sort(order[:max(n, 1)])
        mass = np.cumsum(np.exp(z[kept] - z[order[0]]))
        ids[r] = kept[min(int(np.searchsorted(mass, u[r] * mass[-1], side="right")), len(kept) - 1)]
    return {"output0": torch.from_numpy(ids)}


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    if c["kind"] == "sample":
        return _sample64(c, t) if c["rows"] * c["vocab"] < 4e7 else None
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "window":
        lens = t["lengths"].tolist() if c["padded"] else [c["seq"]] * c["batch"]
        out = torch.zeros((c["batch"], c["seq"], heads, dim), dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            q, k, v = torch.split(t["qkv"][b, :n], [heads, kv, kv], 1)
            out[b, :n] = _attend64(q, k, v, 0, c["window"], c["sinks"])
        return {"output0": out}
    new, lens = _sequences(c)
    table = t["block_tables"].cpu().tolist()
    kc, vc = t["key_cache"], t["value_cache"]
    out, at = [], 0
    if c["kind"] == "append":
        half = c["rotary"] // 2
        kc, vc = kc.double(), vc.double()
        for b in range(c["seqs"]):
            pos = torch.arange(lens[b] - new[b], lens[b], device="cuda")
            z = t["qkv"][at:at + new[b]].double()
            # the pair (i, i + half) as a complex number times e^(i angle)
            turn = torch.complex(t["cos"][pos].double(), t["sin"][pos].double())[:, None]
            pair = torch.complex(z[:, :heads + kv, :half].contiguous(), z[:, :heads + kv, half:2 * half].contiguous()) * turn
            z[:, :heads + kv, :half], z[:, :heads + kv, half:2 * half] = pair.real, pair.imag
            place = torch.tensor(table[b], device="cuda")[pos // c["page"]]
            kc[place, pos % c["page"]], vc[place, pos % c["page"]] = z[:, heads:heads + kv], z[:, heads + kv:]
            out.append(z[:, :heads])
            at += new[b]
        return {"output0": torch.cat(out), "key_cache": kc, "value_cache": vc}
    for b in range(c["seqs"]):
        pages = torch.tensor([x for x in table[b] if x >= 0], device="cuda")
        k, v = (x[pages].reshape(-1, kv, dim)[:lens[b]] for x in (kc, vc))
        out.append(_attend64(t["q"][at:at + new[b]], k, v, lens[b] - new[b], c["window"], c["sinks"]))
        at += new[b]
    return {"output0": torch.cat(out)}
