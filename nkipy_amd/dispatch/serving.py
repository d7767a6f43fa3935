"""Lowering of the serving operators (``nkipy_amd.core.ops.serving``): their
launch helpers and the patterns that claim their nodes.

Operands are read in place through the strides of the views they were taken
by (heads sliced out of a projection, transposed tensors).  ``rotary_append``
traces to one node per result (the rotated q, each cache); they become one
launch.  A cache that is an argument of the kernel is written in its own
buffer, rows of other positions staying as they are.
"""

from __future__ import annotations

import ctypes
from typing import Dict, List, Tuple

import numpy as np

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core.backend.ir import Node, Value
from nkipy_amd.dispatch import generic as G
from nkipy_amd.dispatch.launchers import Launch, LaunchError, dtype_tag
from nkipy_amd.dispatch.patterns import LaunchStep, Match
from nkipy_amd.dispatch.plan import Slot
from nkipy_amd.dispatch.views import View, resolve

NO_WINDOW = 2**30


# ---------------------------------------------------------------------------
# Launch helpers
# ---------------------------------------------------------------------------
class AppendArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "oq", "ok", "ov", "cos", "sin", "tables", "lens",
                                                 "starts")]
                + [(n, ctypes.c_int64) for n in ("q_ss", "q_sh", "k_ss", "k_sh", "v_ss", "v_sh")]
                + [(n, ctypes.c_int32) for n in ("B", "N", "Hq", "Hkv", "D", "half", "P", "page", "pages", "width")])


class AttendArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "tables", "lens", "starts", "first", "ws", "zeros")]
                + [(n, ctypes.c_int64) for n in ("q_sb", "q_ss", "q_sh", "k_sb", "k_ss", "k_sh", "v_sb", "v_ss", "v_sh")]
                + [(n, ctypes.c_int32) for n in ("B", "S", "N", "T", "Hq", "Hkv", "D", "page", "pages", "width", "pitch",
                                                 "window", "sinks", "nsplit", "min_blocks", "tiles")]
                + [("scale", ctypes.c_float)])


class SampleArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "u", "out", "temp", "topk", "topp", "minp", "tops", "hist",
                                                 "order", "places", "subs")]
                + [("ld", ctypes.c_int64), ("c_topp", ctypes.c_double)]
                + [(n, ctypes.c_int32) for n in ("rows", "vocab", "seg", "nseg", "sub")]
                + [("c_temp", ctypes.c_float), ("c_topk", ctypes.c_int32), ("c_minp", ctypes.c_float)])


def _fields(args, **values):
    for n, x in values.items():
        setattr(args, n, x)
    return args


def rotary_append(dtype, B, N, Hq, Hkv, D, half, P, page, pages, width, *, q=0, k=0, v=0, oq=0, ok=0, ov=0, cos=0, sin=0,
                  tables=0, lens=0, starts=0, q_str=(0, 0), k_str=(0, 0), v_str=(0, 0)) -> Launch:
    """Rotates q into oq and k into the cache ok, copies v into the cache ov;
    parts whose output is null are left out.  Strides are (row, head)."""
    if N < 1 or B < 1 or N >= 2**31 or B >= 2**31:
        raise LaunchError(f"rotary_append: {N} tokens of {B} sequences")
    if (oq or ok) and not 0 < 2 * half <= D:
        raise LaunchError(f"rotary_append: {2 * half} rotated elements of {D}")
    if not oq and not ok:
        half = 0  # values only
    if (ok or ov) and not (tables and page > 0 and pages > 0 and width > 0):
        raise LaunchError("rotary_append: a cache needs its block table")
    a = _fields(AppendArgs(), q=q, k=k, v=v, oq=oq, ok=ok, ov=ov, cos=cos, sin=sin, tables=tables, lens=lens, starts=starts,
                q_ss=q_str[0], q_sh=q_str[1], k_ss=k_str[0], k_sh=k_str[1], v_ss=v_str[0], v_sh=v_str[1],
                B=B, N=N, Hq=Hq if oq else 0, Hkv=Hkv, D=D, half=half, P=P, page=max(page, 1), pages=pages, width=width)
    size = dt.itemsize(dtype)
    # pieces of eight elements: whole, and at 16-byte addresses
    whole = half % 8 == 0 and D % 8 == 0 and not any(p % 16 for p in (q, k, v, oq, ok, ov, cos, sin)) \
        and not any(s * size % 16 for s in q_str + k_str + v_str)
    nbytes = 2 * size * N * D * ((Hq if oq else 0) + (Hkv if ok else 0) + (Hkv if ov else 0)) + 8 * N * half
    return Launch("serving", f"nk_rotary_append{'' if whole else '1'}_{dtype_tag(dtype)}", (N, 1, 1), (256, 1, 1), a,
                  bytes=nbytes)


ATT_ROWS, ATT_KEYS = 128, 32  # rows of a tile, keys of a block (attend_index.h)
ATT_CUS, ATT_SLOTS = 256, 512  # CUs; workgroups that a step is split into (two a CU; three or more would fit)
ATT_STEP_GRID = 2048          # workgroups of a step, to even out lengths
ATT_STEP_BLOCKS = 32          # blocks that a split of a step has at least past ATT_SLOTS
ATT_MIN_BLOCKS = 4            # blocks that any split of a step has at least
ATT_TILE_BLOCKS = 8           # blocks that a tile's split has at least
ATT_MAX_SPLIT = 64            # a lane of the joining wave for each
ATT_JOIN_WIDE = 4             # splits past which a workgroup joins a row of fewer
ATT_JOIN_ROWS = 1024          # than this; a wave does it where waves fill the chip
ATT_STEP_HEADS = 16           # heads of a group in one workgroup of a step


def attend_tiled(dtype, D) -> bool:
    """Whether the tiled and step kernels have this type and head dim."""
    return dt.canonical(dtype) in (dt.bfloat16, dt.float16) and D in (64, 128)


def attend_work(B, S, N, Hq, Hkv, D, keys, window=0, sinks=0, starts=False) -> Tuple[bool, int, int]:
    """(whether this is a step, workgroups of a KV head and split, splits of the
    keys): one new token per sequence is a step.  Splits are for the longest
    sequence that the tensors can hold; the kernels give a shorter one fewer.

    A step's keys are split where the rest leaves CUs idle, and long ones
    further, so that sequences of many lengths end together (64 of up to 8192
    keys: 263 us with one split, 242 with four; 64 with a window of 500: 27 us
    with one, 33 with four).

    Tiles take the splits of the least estimate: a block of keys counts 0.75 for
    a CU's only workgroup and 0.52 for each of more; the sums of every split are
    written and read at 4.5 TB/s, by a launch of 5.  The constants were fitted, at
    head dim 128, to which split wins below; they rank splits and are no times
    (2100 tokens of 24 sequences in a window of 1024: 55 by the estimate, 82 us
    measured, as two workgroups share a CU and the third waits).  Measured, whole
    calls: 1000 tokens of one prompt 27 us with one split, 46 with eight; 256
    tokens behind 3744 cached 42 with seven or four, 95 with one; 40 tokens of
    eight sequences of 8000 44 with seven, 72 with three; the 2100 tokens 82 with
    one, 115 with two."""
    rep = Hq // Hkv
    step = not starts and S == 1
    if step:
        units, tokens = B * -(-rep // ATT_STEP_HEADS), 1
    else:
        units = N * rep // ATT_ROWS + B if starts else B * -(-S * rep // ATT_ROWS)
        tokens = -(-ATT_ROWS // rep)
    seen = min(keys, window + sinks + tokens + ATT_KEYS) if window else keys
    blocks = -(-seen // ATT_KEYS)
    if step:
        splits = ATT_SLOTS // (units * Hkv)
        splits = max(splits, min(ATT_STEP_GRID // (units * Hkv), seen // (ATT_KEYS * ATT_STEP_BLOCKS)))
        splits = min(splits, -(-blocks // ATT_MIN_BLOCKS))
    else:
        def cost(s):
            join = 5 + s * N * Hq * (D + 2) * 8 / 4.5e6 if s > 1 else 0
            return -(-blocks // s) * max(0.75, 0.52 * -(-units * Hkv * s // ATT_CUS)) + join
        splits = min(range(1, min(ATT_MAX_SPLIT, max(1, blocks // ATT_TILE_BLOCKS)) + 1), key=cost)
    return step, units, max(1, min(splits, ATT_MAX_SPLIT))


def attend_join(dtype, a: AttendArgs) -> Launch:
    """The launch that joins the splits of ``a``.  Whole calls with a workgroup
    a row and with a wave, us: 32 rows of 63 splits 14.4 and 31.5, of 12 10.2
    and 10.5, 256 of 19 97 and 100, 1280 of 7 45.5 and 43.8."""
    rows, tag = a.N * a.Hq, f"{dtype_tag(dtype)}_d{a.D}"
    if a.nsplit > ATT_JOIN_WIDE and rows < ATT_JOIN_ROWS:
        return Launch("attend", f"nk_attend_join4_{tag}", (rows, 1, 1), (256, 1, 1), a)
    return Launch("attend", f"nk_attend_join_{tag}", (-(-rows // 4), 1, 1), (256, 1, 1), a)


def attend(dtype, q, k, v, o, *, B, N, Hq, Hkv, D, q_str, k_str, v_str, scale, S=1, T=0, tables=0, lens=0, starts=0, first=0,
           page=1, pages=0, width=0, pitch=0, window=0, sinks=0, ws=0, zeros=0) -> List[Launch]:
    """Attention over a paged cache (``tables``; strides of q are (0, row,
    head), of the cache (0, row, head) with ``pitch`` rows from page to page)
    or plain tensors (B sequences of S queries and T keys; strides (sequence,
    row, head)).  ``zeros``: D zeros of the operands' type, for the tiled form;
    ``ws``: 4 splits N Hq (D + 2) bytes where ``attend_work`` splits."""
    if N < 1 or B < 1 or N * Hq >= 2**31:
        raise LaunchError(f"attention of {N} queries of {B} sequences and {Hq} heads")
    if Hkv < 1 or Hq % Hkv or not 1 <= D <= 256:
        raise LaunchError(f"attention: {Hq} / {Hkv} heads of {D}")
    if tables:
        if width < 1 or page < 1 or width * page >= 2**30 or pages * pitch >= 2**31:
            raise LaunchError("attention: cache too large, or no page")
        if pitch < page:
            raise LaunchError(f"attention: pages of {page} rows at a pitch of {pitch}")
    elif B * S != N or T >= 2**30 or S >= 2**30:
        raise LaunchError("attention: sequences too long")
    if min(k_str[1], v_str[1]) < (1 if tables else 0):
        raise LaunchError(f"attention: row strides {k_str[1]} and {v_str[1]} of keys and values")
    a = _fields(AttendArgs(), q=q, k=k, v=v, o=o, tables=tables, lens=lens, starts=starts, first=first,
                q_sb=q_str[0], q_ss=q_str[1], q_sh=q_str[2], k_sb=k_str[0], k_ss=k_str[1], k_sh=k_str[2],
                v_sb=v_str[0], v_ss=v_str[1], v_sh=v_str[2], B=B, S=S, N=N, T=T, Hq=Hq, Hkv=Hkv, D=D, page=page, pages=pages,
                width=width, pitch=pitch, window=window or NO_WINDOW, sinks=sinks, nsplit=1, min_blocks=1, scale=scale,
                ws=ws, zeros=zeros)
    tag = dtype_tag(dtype)
    tiled = attend_tiled(dtype, D) and zeros and not any(x % 16 for x in (q, k, v, o, zeros, ws)) \
        and not any(x % 8 for x in (*q_str, *k_str, *v_str))
    if not tiled:
        return [Launch("attend", f"nk_attend_rows_{tag}", (-(-N * Hq // 4), 1, 1), (256, 1, 1), a)]
    step, a.tiles, a.nsplit = attend_work(B, S, N, Hq, Hkv, D, width * page if tables else T, window, sinks, bool(starts))
    a.min_blocks = ATT_MIN_BLOCKS if step else ATT_TILE_BLOCKS
    if a.nsplit > 1 and not ws:
        raise LaunchError(f"attention of {a.nsplit} splits needs a workspace")
    if a.tiles * Hkv * a.nsplit >= 2**31 or Hq // Hkv * S >= 2**31:
        raise LaunchError("attention: too many tiles for one launch")
    # tiles address a sequence's rows by 32-bit offsets where those reach
    reach = 2 * max(k_str[1], v_str[1]) * (pages * pitch if tables else T + 64)
    far = not step and (reach >= 2**32 - 4096 or (tables and k_str[1] != v_str[1]))
    kind = f"{'step' if step else 'tile'}_{'paged' if tables else 'plain'}{'_far' if far else ''}"
    out = [Launch("attend", f"nk_attend_{kind}_{tag}_d{D}", (a.tiles * Hkv * a.nsplit, 1, 1), (256, 1, 1), a)]
    if a.nsplit > 1:
        out.append(attend_join(dtype, a))
    return out


# tokens of a row in one launch, bins of a histogram, parts of a row (serving.hip)
SMP_LIST, SMP_BINS, SMP_SUBS = 8192, 512, 1024


def sample_segments(rows: int, vocab: int) -> Tuple[int, int]:
    """(tokens of a segment, segments of a row): as long as the segments still
    fill the CUs, since the last launch adds a histogram for each."""
    for seg in (8192, 4096, 2048):
        if seg == 2048 or rows * -(-vocab // seg) >= 512:
            break
    while -(-vocab // seg) > 1024:
        seg *= 2
    return seg, -(-vocab // seg)


def sample_parts(nseg: int) -> int:
    """Parts of a segment whose largest values are kept: up to 64, of 4 to 64
    lanes each, and up to SMP_SUBS in a row; 0 where there are more segments."""
    sub = 64
    while sub >= 4 and nseg * sub > SMP_SUBS:
        sub //= 2
    return sub if sub >= 4 else 0


def sample_workspace_bytes(rows: int, vocab: int) -> int:
    if vocab <= SMP_LIST:
        return 0
    seg, nseg = sample_segments(rows, vocab)
    return rows * nseg * (8 * (SMP_BINS + 2) + 2 * (seg + SMP_BINS + 2 + sample_parts(nseg)))


def sample(dtype, x, u, out, rows, vocab, ld, *, temperature, top_k, top_p, min_p, ws=0) -> List[Launch]:
    """One token per row of logits; each filter is (address of one value per
    row or 0, number).  ``ws``: ``sample_workspace_bytes``."""
    if rows < 1 or not 1 <= vocab <= 2**22:
        raise LaunchError(f"sample: {rows} rows of {vocab}")
    a = _fields(SampleArgs(), x=x, u=u, out=out, ld=ld, rows=rows, vocab=vocab, temp=temperature[0],
                # (above 0 in 32 bits too: 0 is the largest logit's)
                c_temp=max(temperature[1], 2.0**-149) if temperature[1] > 0 else 0.0,
                topk=top_k[0], c_topk=top_k[1], topp=top_p[0], c_topp=top_p[1], minp=min_p[0], c_minp=min_p[1])
    tag, nbytes = dtype_tag(dtype), rows * (vocab * dt.itemsize(dtype) + 8)
    if vocab <= SMP_LIST:
        return [Launch("serving", f"nk_sample_row_{tag}", (rows, 1, 1), (1024, 1, 1), a, bytes=nbytes)]
    a.seg, a.nseg = sample_segments(rows, vocab)
    if not ws or ws % 8:
        raise LaunchError("sample: long rows need a workspace")
    n = -(-rows // 8) * 8 * a.nseg
    if n >= 2**31:
        raise LaunchError("sample: too many rows for one launch")
    every = rows * a.nseg
    order = ws + 8 * every * (SMP_BINS + 2)
    places = order + 2 * every * a.seg
    _fields(a, sub=sample_parts(a.nseg), tops=ws, hist=ws + 8 * every, order=order, places=places,
            subs=places + 2 * every * (SMP_BINS + 2))
    return [Launch("serving", f"nk_sample_top_{tag}", (n, 1, 1), (256, 1, 1), a, bytes=nbytes),
            Launch("serving", f"nk_sample_hist_{tag}", (n, 1, 1), (256, 1, 1), a, bytes=nbytes),
            Launch("serving", f"nk_sample_pick_{tag}", (rows, 1, 1), (1024, 1, 1), a)]


# ---------------------------------------------------------------------------
# Operand views
# ---------------------------------------------------------------------------
def _contiguous(v: Value) -> Tuple[View, List[int]]:
    vw = View(v, 0, [])
    return vw, G.contiguous_strides(v.shape)


def _strided(v: Value) -> Tuple[View, List[int]]:
    """``v`` as a view with one stride per dimension and a dense last one, or
    ``v`` itself, materialised: a step of its own in the plan, which copies all of
    it (a cache whose layout is no such view is better laid out once)."""
    vw = resolve(v, widen_ok=False)
    st = [vw.simple(d) for d in range(v.ndim)]
    if any(s is None for s in st) or (st[-1] != 1 and v.shape[-1] != 1) or vw.base.dtype != v.dtype:
        return _contiguous(v)
    return vw, st


def _cache_strided(v: Value):
    """A cache (pages, page, heads, dim) whose pages lie a whole number of rows
    apart, at least a page's own (the tiles' buffer resource ends behind the last
    of them): (view, (0, row, head), rows from page to page)."""
    vw, st = _strided(v)
    pages, page = v.shape[:2]
    if page == 1:
        st[1] = st[0] if pages > 1 else max(st[0], 1)
    if pages == 1:
        st[0] = st[1] * page
    if st[1] < 1 or st[0] < st[1] * page or st[0] % st[1] or st[0] // st[1] * pages >= 2**31:
        vw, st = _contiguous(v)
    return vw, (0, st[1], st[2]), st[0] // st[1]


def _at(addr, vw: View) -> int:
    return addr(vw.base) + vw.offset * vw.base.dtype.itemsize


# ---------------------------------------------------------------------------
# Patterns
# ---------------------------------------------------------------------------
class AppendMatch(Match):
    """The nodes of one ``rotary_append``: one launch."""

    name = "rotary_append"

    def __init__(self, nodes: List[Node]):
        self.parts: Dict[str, Node] = {}
        for n in nodes:
            self.parts["q" if n.op == "rotate_rows" else "k" if n.attrs["rotary"] else "v"] = n
        self.views = {p: _strided(n.inputs[0 if p == "q" else 1]) for p, n in self.parts.items()}
        inputs = []
        for p, n in self.parts.items():
            rest = n.inputs[1:] if p == "q" else [n.inputs[0]] + n.inputs[2:]
            inputs += [self.views[p][0].base] + rest
        super().__init__(nodes, list(dict.fromkeys(inputs)), [n.out for n in nodes])

    def steps(self, plan):
        parts, views = self.parts, self.views
        steps, shape = [], {}
        for p in ("k", "v"):
            if p not in parts:
                continue
            n = parts[p]
            cache = n.inputs[0]
            shape = dict(page=cache.shape[1], pages=cache.shape[0], Hkv=cache.shape[2], D=cache.shape[3])
            # the caller's buffer (behind an earlier write, too), or a copy of the cache
            # where that is still read
            src, dst = plan.buffers[plan.slot(cache).buffer], plan.buffers[plan.slot(n.out).buffer]
            own = src is dst or dst.kind == "output" and src.kind == "input" and plan.alias_outputs.get(dst.name) == src.name
            if not own:
                steps.append(G.ProgramStep(f"copy {cache!r}", G.flat_copy_program(cache), n.out))
        some = next(iter(parts.values()))
        starts = some.inputs[-1] if some.attrs["starts"] else None
        lens = some.inputs[-2 if starts is not None else -1]
        table = next((n.inputs[4 if n.attrs["rotary"] else 2] for p, n in parts.items() if p != "q"), None)
        cos = next((n.inputs[1 if p == "q" else 2] for p, n in parts.items() if p != "v"), None)
        sin = next((n.inputs[2 if p == "q" else 3] for p, n in parts.items() if p != "v"), None)
        rows = some.inputs[0 if some.op == "rotate_rows" else 1]
        if "q" in parts:
            q = parts["q"].inputs[0]
            shape = {"page": 1, "pages": 0, "Hkv": 0, **shape, "Hq": q.shape[1], "D": q.shape[2]}
        # (values alone have no tables, and still drop what has no row in them)
        P, half = cos.shape if cos is not None else (some.attrs["positions"], 0)

        def make(addr):
            kw = {}
            for p, n in parts.items():
                vw, st = views[p]
                kw.update({p: _at(addr, vw), "o" + p: addr(n.out), p + "_str": (st[0], st[1])})
            if table is not None:
                kw.update(tables=addr(table), width=table.shape[1])
            if cos is not None:
                kw.update(cos=addr(cos), sin=addr(sin))
            return rotary_append(rows.dtype, lens.shape[0], rows.shape[0], lens=addr(lens),
                                 starts=addr(starts) if starts is not None else 0, half=half, P=P,
                                 **{**dict(Hq=0, width=0), **shape, **kw})

        if rows.size:
            desc = f"rotary append {rows.shape[0]} tokens of {lens.shape[0]} sequences: {', '.join(sorted(parts))}"
            steps.append(LaunchStep("rotary_append", desc, self.inputs, self.outputs, make))
        return steps


class AppendPattern:
    def find(self, L):
        group: List[Node] = []
        for n in L.live + [None]:
            if n is not None and n.op in ("rotate_rows", "paged_write"):
                if group and not self._joins(group, n):
                    yield from self._claim(L, group)
                    group = []
                group.append(n)
                continue
            # the nodes of a call follow each other in the trace
            if group:
                yield from self._claim(L, group)
                group = []

    @staticmethod
    def _shared(n: Node):
        """What the parts of one launch have in common, by name."""
        where = n.inputs[-(1 + n.attrs["starts"]):]
        rows = n.inputs[0 if n.op == "rotate_rows" else 1]
        out = {"where": [v.id for v in where], "rows": (rows.shape[0], rows.shape[2], rows.dtype)}
        if n.op == "rotate_rows" or n.attrs["rotary"]:
            at = 1 if n.op == "rotate_rows" else 2
            out["turn"] = [v.id for v in n.inputs[at:at + 2]]
            out["positions"] = n.inputs[at].shape[0]
        else:
            out["positions"] = n.attrs["positions"]
        if n.op == "paged_write":
            out["cache"] = (n.inputs[0].shape, n.inputs[4 if n.attrs["rotary"] else 2].id)
        return out

    def _joins(self, group, n):
        kind = lambda m: (m.op, m.attrs.get("rotary"))  # noqa: E731
        mine = self._shared(n)
        return all(kind(m) != kind(n) and all(mine.get(x, y) == y for x, y in self._shared(m).items()) for m in group)

    @staticmethod
    def _claim(L, group):
        m = AppendMatch(group)
        # (a cache written twice, or q computed from a cache written here, is
        # no single launch)
        outs = {n.out.id for n in group}
        if not any(v.id in outs for v in m.inputs) and m.validate(L):
            yield m
            return
        for n in group:
            one = AppendMatch([n])
            if one.validate(L):
                yield one


class AttendMatch(Match):
    """``paged_attention`` or ``window_attention``."""

    name = "attend"

    def __init__(self, n: Node):
        self.node, self.paged = n, n.op == "paged_attention"
        q, k, v = n.inputs[:3]
        self.q, self.q_str = _strided(q)
        if self.paged:
            (self.k, self.k_str, self.pitch), (self.v, self.v_str, vp) = _cache_strided(k), _cache_strided(v)
            if vp != self.pitch:  # one row number serves both
                (self.k, ks), (self.v, vs) = _contiguous(k), _contiguous(v)
                self.k_str, self.v_str, self.pitch = (0, ks[1], ks[2]), (0, vs[1], vs[2]), k.shape[1]
            self.q_str = [0] + list(self.q_str[:2])
        else:
            (self.k, ks), (self.v, vs) = _strided(k), _strided(v)
            self.q_str, self.k_str, self.v_str, self.pitch = self.q_str[:3], ks[:3], vs[:3], 0
        super().__init__([n], list(dict.fromkeys([self.q.base, self.k.base, self.v.base] + n.inputs[3:])), [n.out])

    def steps(self, plan):
        n, at = self.node, self.node.attrs
        q, k = n.inputs[:2]
        kw = dict(window=at["window"], sinks=at["sinks"], scale=at["scale"], q_str=self.q_str, k_str=self.k_str,
                  v_str=self.v_str, Hq=q.shape[-2], Hkv=k.shape[2], D=q.shape[-1])
        more = {}
        if self.paged:
            tables = n.inputs[3]
            kw.update(B=tables.shape[0], N=q.shape[0], page=k.shape[1], pages=k.shape[0], width=tables.shape[1],
                      pitch=self.pitch)
            more = dict(tables=tables, lens=n.inputs[4])
            if at["starts"]:
                more["starts"] = n.inputs[5]
        else:
            kw.update(B=q.shape[0], S=q.shape[1], N=q.shape[0] * q.shape[1], T=k.shape[1])
            rest = list(n.inputs[3:])
            if at["lengths"]:
                more["lens"] = rest.pop(0)
            if at["positions"]:
                more["first"] = rest.pop(0)
        if not q.size:
            return []
        tmp = {}
        if attend_tiled(q.dtype, kw["D"]):
            keys = tables.shape[1] * k.shape[1] if self.paged else k.shape[1]
            splits = attend_work(kw["B"], kw.get("S", 1), kw["N"], kw["Hq"], kw["Hkv"], kw["D"], keys, kw["window"], kw["sinks"],
                                 "starts" in more)[2]
            tmp["zeros"] = Slot(plan.add_buffer(2 * kw["D"], "const", "attend.zeros", np.zeros(kw["D"], np.uint16)))
            if splits > 1:
                tmp["ws"] = Slot(plan.add_buffer(4 * splits * kw["N"] * kw["Hq"] * (kw["D"] + 2), "temp", "attend.splits"))

        def make(addr):
            return attend(q.dtype, _at(addr, self.q), _at(addr, self.k), _at(addr, self.v), addr(n.out),
                          **kw, **{x: addr(y) for x, y in {**more, **tmp}.items()})

        desc = (f"{'paged' if self.paged else 'window'} attention N={kw['N']} B={kw['B']} Hq={kw['Hq']} Hkv={kw['Hkv']} "
                f"D={kw['D']} window={at['window']} sinks={at['sinks']}")
        return [LaunchStep("attend", desc, self.inputs, self.outputs, make)]


class SampleMatch(Match):
    name = "sample"

    def __init__(self, n: Node):
        self.node = n
        x = n.inputs[0]
        vw, st = _strided(x)
        self.x, self.ld = vw, st[0]
        super().__init__([n], list(dict.fromkeys([vw.base] + n.inputs[1:])), [n.out])

    def steps(self, plan):
        n = self.node
        rows, vocab = n.inputs[0].shape
        if not rows:
            return []
        given, rest = {}, list(n.inputs[2:])
        for name, none in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)):
            x = n.attrs.get(name)
            given[name] = (rest.pop(0), none) if x == "rows" else (None, none if x is None else x)

        need = sample_workspace_bytes(rows, vocab)
        ws = Slot(plan.add_buffer(need, "temp", "sample.segments")) if need else None

        def make(addr):
            f = {name: (addr(v) if v is not None else 0, c) for name, (v, c) in given.items()}
            return sample(n.inputs[0].dtype, _at(addr, self.x), addr(n.inputs[1]), addr(n.out), rows, vocab, self.ld,
                          ws=addr(ws) if ws is not None else 0, **f)

        return [LaunchStep("sample", f"sample {rows}x{vocab}", self.inputs, self.outputs, make)]


class ServingPattern:
    """The attentions and the draw: one node each."""

    KINDS = {"paged_attention": AttendMatch, "window_attention": AttendMatch, "sample": SampleMatch}

    def find(self, L):
        for n in L.live:
            kind = self.KINDS.get(n.op)
            if kind is not None and id(n) not in L.covered:
                m = kind(n)
                if m.validate(L):
                    yield m
