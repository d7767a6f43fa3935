"""Lowering of the paged cache of 8-bit codes (``nkipy_amd.core.ops.serving_fp8``):
launch helpers and patterns.

Queries and the rows to append are read in place through the strides of the
views they were taken by; the caches and exponents of an append are written in
the caller's buffers.  Attention takes the tiles, splits and joining launches of
the attention over 16-bit caches.
"""

from __future__ import annotations

import ctypes
from typing import List, Tuple

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core.backend.ir import Node
from nkipy_amd.dispatch import serving as S
from nkipy_amd.dispatch.beams import UpdateMatch, calls
from nkipy_amd.dispatch.launchers import Launch, LaunchError, dtype_tag
from nkipy_amd.dispatch.patterns import LaunchStep, Match
from nkipy_amd.dispatch.plan import Slot
from nkipy_amd.dispatch.serving import _at, _cache_strided, _contiguous, _fields, _strided


# ---------------------------------------------------------------------------
# Launch helpers
# ---------------------------------------------------------------------------
class Append8Args(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "v", "oq", "kc", "vc", "ke", "ve", "cos", "sin", "tables", "lens",
                                                 "starts")]
                + [(n, ctypes.c_int64) for n in ("q_ss", "q_sh", "k_ss", "k_sh", "v_ss", "v_sh")]
                + [(n, ctypes.c_int32) for n in ("B", "N", "Hq", "Hkv", "D", "half", "P", "page", "pages", "width", "heads",
                                              "blocks", "qwaves")])


class Attend8Args(S.AttendArgs):
    _fields_ = [(n, ctypes.c_void_p) for n in ("ke", "ve")]


APPEND_HEADS = 64      # heads of a workgroup at most (append8.hip)
APPEND_ELEMENTS = 2**14  # elements that a workgroup quantises, about
# Tokens from which on a token's queries are one wave's work, not four's (us: 8 tokens of
# 128 heads of 256 10.9 by one wave and 7.0 by four, of 32 of 128 7.3 and 7.1; 2048 of 32
# 23.3 and 25.7, of 64 29.1 and 28.8).
APPEND_TOKENS = 1024


def rotary_append_fp8(dtype, B, N, Hq, Hkv, D, half, P, page, pages, width, *, q, k, v, oq, kc, vc, ke, ve, cos, sin, tables, lens,
                      starts=0, q_str=(0, 0), k_str=(0, 0), v_str=(0, 0)) -> Launch:
    """Rotates q into oq (0: left out), k and v into caches of codes kc / vc
    with exponents ke / ve.  Strides are (row, head)."""
    if N < 1 or B < 1 or N >= 2**31 or B >= 2**30:
        raise LaunchError(f"rotary_append_fp8: {N} tokens of {B} sequences")
    if not (0 < 2 * half <= D and Hkv >= 1 and page >= 1 and pages >= 1 and width >= 1 and pages * page < 2**31
            and width * page < 2**30 and page * D < 2**31):
        raise LaunchError(f"rotary_append_fp8: {2 * half} rotated elements of {D}, {pages} pages of {page}")
    rows = min(page, N) if starts else 1
    heads = max(1, min(Hkv, APPEND_HEADS, APPEND_ELEMENTS // (rows * D)))
    a = _fields(Append8Args(), q=q, k=k, v=v, oq=oq, kc=kc, vc=vc, ke=ke, ve=ve, cos=cos, sin=sin, tables=tables, lens=lens,
                starts=starts, q_ss=q_str[0], q_sh=q_str[1], k_ss=k_str[0], k_sh=k_str[1], v_ss=v_str[0], v_sh=v_str[1],
                B=B, N=N, Hq=Hq, Hkv=Hkv, D=D, half=half, P=P, page=page, pages=pages, width=width, heads=heads)
    blocks = (N // page + 2 * B if starts else B) * 2 * -(-Hkv // heads)
    a.qwaves = 1 if N >= APPEND_TOKENS else 4
    n = (-(-N * a.qwaves // 4) if oq else 0) + blocks
    if n >= 2**31:
        raise LaunchError("rotary_append_fp8: too many workgroups for one launch")
    a.blocks = blocks
    size = dt.itemsize(dtype)
    # pieces of eight elements: whole, and at 16-byte addresses (codes: 8)
    whole = half % 8 == 0 and D % 8 == 0 and not any(x % 16 for x in (q, k, v, oq, kc, vc, cos, sin)) \
        and not any(s * size % 16 for s in (*q_str, *k_str, *v_str))
    nbytes = N * D * (2 * size * (Hq if oq else 0) + 2 * (size + 1) * Hkv) + 8 * N * half
    return Launch("append8", f"nk_append8{'' if whole else '1'}_{dtype_tag(dtype)}", (n, 1, 1), (256, 1, 1), a, bytes=nbytes)


ATT8_WAVES = 4608  # waves that a step is split into where its tables are full: 1.5 times what fits
ATT8_JOIN = 256    # pieces that are joined at most (attend8.hip)


def attend8_work(B, N, Hq, Hkv, D, keys, window=0, sinks=0, starts=False) -> Tuple[bool, int, int, int]:
    """(whether this is a step, its waves or the tiles of a KV head, splits of
    the keys, blocks that a split has at least).

    The pieces of a step have a length, not a number, so that short sequences
    have few and, where the tables are about as wide as the longest sequence, all
    waves end together; their number is a multiple of eight, with which the
    pieces of every sequence come to all XCDs (64 sequences of 400 to 8192 keys,
    whose sums differ by 13% over the XCDs otherwise: 145 us in turns of
    sequences, 121 so).

    The lengths are not known here: pieces and splits follow the tables' width.
    Wider tables have longer pieces (those 64 sequences in tables of 8192, 32768
    and 131072 keys: 119, 288 and 495 us) and more splits of the tiles (2100 tokens
    of 24 sequences of up to 6000, in tables of 6000, 32768 and 131072: 181, 257
    and 257).  The splits of the tiles are weighed by ``attend_work``'s costs of a
    block, which are those of the tiles over 16-bit caches."""
    if starts:
        return S.attend_work(B, 1, N, Hq, Hkv, D, keys, window, sinks, True) + (S.ATT_TILE_BLOCKS,)
    units = B * Hkv * -(-(Hq // Hkv) // S.ATT_STEP_HEADS)
    seen = min(keys, window + sinks + 1 + S.ATT_KEYS) if window else keys
    blocks = -(-seen // S.ATT_KEYS)
    piece = max(1, blocks * units // ATT8_WAVES, -(-blocks // ATT8_JOIN))
    splits = -(-blocks // piece)
    return True, units, -(-splits // 8) * 8 if splits > 1 else 1, piece


def attend8(dtype, q, k, v, o, *, B, N, Hq, Hkv, D, q_str, k_str, v_str, scale, tables, lens, ke, ve, page, pages, width, pitch,
            starts=0, window=0, sinks=0, ws=0) -> List[Launch]:
    """Attention over a paged cache of codes; strides as those of ``attend``
    (those of the cache in bytes, one to an element), workspace as its."""
    if N < 1 or B < 1 or N * Hq >= 2**31:
        raise LaunchError(f"attention of {N} queries of {B} sequences and {Hq} heads")
    if Hkv < 1 or Hq % Hkv or not 1 <= D <= 256:
        raise LaunchError(f"attention: {Hq} / {Hkv} heads of {D}")
    if width < 1 or pages < 1 or page < 1 or width * page >= 2**30 or pages * pitch >= 2**31 or pitch < page:
        raise LaunchError("attention: cache too large, or no page")
    if min(k_str[1], v_str[1]) < 1:
        raise LaunchError(f"attention: row strides {k_str[1]} and {v_str[1]} of keys and values")
    a = _fields(Attend8Args(), q=q, k=k, v=v, o=o, tables=tables, lens=lens, starts=starts, q_ss=q_str[1], q_sh=q_str[2],
                k_ss=k_str[1], k_sh=k_str[2], v_ss=v_str[1], v_sh=v_str[2], B=B, S=1, N=N, Hq=Hq, Hkv=Hkv, D=D, page=page,
                pages=pages, width=width, pitch=pitch, window=window or S.NO_WINDOW, sinks=sinks, nsplit=1, min_blocks=1,
                scale=scale, ws=ws, ke=ke, ve=ve)
    tag = dtype_tag(dtype)
    tiled = S.attend_tiled(dtype, D) and not any(x % 16 for x in (q, k, v, o, ws)) and not any(x % 8 for x in q_str) \
        and not any(x % 16 for x in (*k_str, *v_str))
    if not tiled:
        return [Launch("attend8", f"nk_attend8_rows_{tag}", (-(-N * Hq // 4), 1, 1), (256, 1, 1), a)]
    step, units, a.nsplit, a.min_blocks = attend8_work(B, N, Hq, Hkv, D, width * page, window, sinks, bool(starts))
    a.tiles = B if step else units
    if a.nsplit > 1 and not ws:
        raise LaunchError(f"attention of {a.nsplit} splits needs a workspace")
    n = -(-units * a.nsplit // 4) if step else units * Hkv * a.nsplit
    if n >= 2**29:
        raise LaunchError("attention: too many tiles for one launch")
    out = [Launch("attend8", f"nk_attend8_step_{tag}_d{D}", (n, 1, 1), (256, 1, 1), a) if step else
           Launch("attend8_tile", f"nk_attend8_tile_{tag}_d{D}", (n, 1, 1), (256, 1, 1), a)]
    if a.nsplit > 1 and step:
        out.append(Launch("attend8", f"nk_attend8_join_{tag}_d{D}", (N * Hq, 1, 1), (256, 1, 1), a))
    elif a.nsplit > 1:
        j = S.AttendArgs()
        ctypes.memmove(ctypes.addressof(j), ctypes.addressof(a), ctypes.sizeof(j))
        out.append(S.attend_join(dtype, j))
    return out


# ---------------------------------------------------------------------------
# Patterns
# ---------------------------------------------------------------------------
class Append8Match(UpdateMatch):
    name = "rotary_append_fp8"

    def __init__(self, nodes: List[Node]):
        self.views = [_strided(v) for v in nodes[0].inputs[:3]]
        super().__init__(nodes, {i: vw for i, (vw, _) in enumerate(self.views)})

    def steps(self, plan):
        q, k, _, cos, sin, key, _, _, _, tables, lens = self.operands[:11]
        starts = self.operands[11] if self.at["starts"] else None
        steps, to = self.begin(plan, {})
        if not q.size:
            return steps
        pages, page, hkv, dim = key.shape

        def make(addr):
            places = {x: _at(addr, vw) for x, (vw, _) in zip("qkv", self.views)}
            strides = {x + "_str": (st[0], st[1]) for x, (_, st) in zip("qkv", self.views)}
            return rotary_append_fp8(q.dtype, lens.shape[0], q.shape[0], q.shape[1], hkv, dim, cos.shape[1], cos.shape[0], page,
                                     pages, tables.shape[1], oq=addr(to["q"]) if "q" in to else 0, kc=addr(to["key_cache"]),
                                     vc=addr(to["value_cache"]), ke=addr(to["key_exps"]), ve=addr(to["value_exps"]),
                                     cos=addr(cos), sin=addr(sin), tables=addr(tables), lens=addr(lens),
                                     starts=addr(starts) if starts is not None else 0, **places, **strides)

        desc = f"rotary append of codes {q.shape[0]} tokens of {lens.shape[0]} sequences"
        return steps + [LaunchStep("rotary_append_fp8", desc, self.inputs, self.outputs, make)]


class Attend8Match(Match):
    name = "attend8"

    def __init__(self, n: Node):
        self.node = n
        q, k, v = n.inputs[:3]
        self.q, st = _strided(q)
        self.q_str = [0] + list(st[:2])
        (self.k, self.k_str, self.pitch), (self.v, self.v_str, vp) = _cache_strided(k), _cache_strided(v)
        if vp != self.pitch:  # one row number serves both
            (self.k, ks), (self.v, vs) = _contiguous(k), _contiguous(v)
            self.k_str, self.v_str, self.pitch = (0, ks[1], ks[2]), (0, vs[1], vs[2]), k.shape[1]
        super().__init__([n], list(dict.fromkeys([self.q.base, self.k.base, self.v.base] + n.inputs[3:])), [n.out])

    def steps(self, plan):
        n, at = self.node, self.node.attrs
        q, k, _, ke, ve, tables, lens = n.inputs[:7]
        if not q.size:
            return []
        more = dict(tables=tables, lens=lens, ke=ke, ve=ve)
        if at["starts"]:
            more["starts"] = n.inputs[7]
        kw = dict(B=tables.shape[0], N=q.shape[0], Hq=q.shape[1], Hkv=k.shape[2], D=q.shape[2], page=k.shape[1], pages=k.shape[0],
                  width=tables.shape[1], pitch=self.pitch, window=at["window"], sinks=at["sinks"], scale=at["scale"],
                  q_str=self.q_str, k_str=self.k_str, v_str=self.v_str)
        if S.attend_tiled(q.dtype, kw["D"]):
            splits = attend8_work(kw["B"], kw["N"], kw["Hq"], kw["Hkv"], kw["D"], kw["width"] * kw["page"], kw["window"],
                                  kw["sinks"], at["starts"])[2]
            if splits > 1:
                more["ws"] = Slot(plan.add_buffer(4 * splits * kw["N"] * kw["Hq"] * (kw["D"] + 2), "temp", "attend8.splits"))

        def make(addr):
            return attend8(q.dtype, _at(addr, self.q), _at(addr, self.k), _at(addr, self.v), addr(n.out), **kw,
                           **{x: addr(y) for x, y in more.items()})

        desc = (f"paged attention of codes N={kw['N']} B={kw['B']} Hq={kw['Hq']} Hkv={kw['Hkv']} D={kw['D']} "
                f"window={at['window']} sinks={at['sinks']}")
        return [LaunchStep("attend8", desc, self.inputs, self.outputs, make)]


class Fp8CachePattern:
    def find(self, L):
        for group in calls(L, ("append_fp8",)):
            m = Append8Match(group)
            if m.validate(L):
                yield m
        for n in L.live:
            if n.op == "paged_attention_fp8":
                m = Attend8Match(n)
                if m.validate(L):
                    yield m
