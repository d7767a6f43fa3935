"""Lowering of the generation loop's operators (``nkipy_amd.core.ops.beams``)
and the base of matches that update arrays in place.

An operator with several results traces to one node for each, over the same
operands (``serving_fp8.build_updates``); they become the launches of one call.
A launch updates an array where it stands: in the caller's buffer, under the
rule of the other in-place writes, else in a copy of it.
"""

from __future__ import annotations

import ctypes
from typing import Dict, List, Tuple

from nkipy_amd.core import dtypes as dt
from nkipy_amd.core.backend.ir import Node, Value
from nkipy_amd.dispatch import generic as G
from nkipy_amd.dispatch.launchers import Launch, LaunchError, dtype_tag
from nkipy_amd.dispatch.patterns import LaunchStep, Match
from nkipy_amd.dispatch.plan import Slot
from nkipy_amd.dispatch.serving import _at, _fields, _strided
from nkipy_amd.dispatch.views import View

MAX_BEAMS = 32


# ---------------------------------------------------------------------------
# Launch helpers
# ---------------------------------------------------------------------------
class AssignArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("tables", "lens", "news", "starts", "slots", "free", "wants", "list", "marks")]
                + [(n, ctypes.c_int32) for n in ("rows", "width", "page", "pages", "tokens", "parts")])


class SelectArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "scores", "ended", "tokens", "parents", "out", "ends", "sums", "best")]
                + [("ld", ctypes.c_int64)]
                + [(n, ctypes.c_int32) for n in ("groups", "beams", "vocab", "nseg", "end")])


class ReorderArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("parents", "lens", "tables", "k", "v", "ke", "ve")]
                + [("row", ctypes.c_int64)]
                + [(n, ctypes.c_int32) for n in ("groups", "beams", "width", "page", "pages", "hkv", "tblocks", "kblocks")])


ASSIGN_PAGES = 2**20  # bits of a workgroup's LDS
ASSIGN_SMALL = 1024   # tokens, and
ASSIGN_ROWS = 64      # rows, of
ASSIGN_WIDTH = 2048   # entries each, and
ASSIGN_ENTRIES = 2**15  # in all, that one workgroup deals with
ASSIGN_MARKS = 64     # rows that a workgroup marks at once, four a wave
ASSIGN_WORDS = 2**18  # words of bitmaps that one workgroup joins, about


def assign_parts(rows, width, pages, tokens) -> int:
    """Workgroups that mark the pages held, 0 where one does everything (by one
    workgroup and by three launches, us: 64 rows of 250 entries 11.6 and 13.2, of
    512 14.7 and 15.2; 8 of 2048 14.4 and 16.1; 1 of 250 with 1000 tokens 11.6 and
    14.8; 96 of 256 15.3 and 14.1; 1 of 6250 20.8 and 17.7; 16 of 250 with 2048
    tokens 16.3 and 15.0)."""
    if tokens <= ASSIGN_SMALL and rows <= ASSIGN_ROWS and width <= ASSIGN_WIDTH and rows * width <= ASSIGN_ENTRIES:
        return 0
    return max(1, min(-(-rows // ASSIGN_MARKS), ASSIGN_WORDS // -(-pages // 32)))


def assign_workspace_bytes(rows, width, pages, tokens) -> int:
    return 16 * (-(-rows // 4) + -(-pages // 4) + assign_parts(rows, width, pages, tokens) * -(-pages // 128))


def assign_pages(rows, width, page, pages, tokens, *, tables, lens, news, starts, slots, free, ws) -> List[Launch]:
    """Tables updated in place, starts (rows + 1), slots (tokens) and the
    number of pages left; ``ws``: ``assign_workspace_bytes``."""
    if not (1 <= rows <= 2**16 and width >= 1 and 1 <= pages <= ASSIGN_PAGES and page >= 1 and 0 <= tokens <= 2**30
            and width * page < 2**30 and pages * page < 2**31):
        raise LaunchError(f"assign_pages: {tokens} tokens of {rows} rows of {width}, {pages} pages of {page}")
    parts = assign_parts(rows, width, pages, tokens)
    taken = ws + 16 * -(-rows // 4)
    a = _fields(AssignArgs(), tables=tables, lens=lens, news=news, starts=starts, slots=slots, free=free, wants=ws, list=taken,
                marks=taken + 16 * -(-pages // 4), rows=rows, width=width, page=page, pages=pages, tokens=tokens, parts=parts)
    if not parts:
        return [Launch("beams", "nk_assign_pages", (1, 1, 1), (1024, 1, 1), a)]
    return [Launch("beams", "nk_assign_mark", (parts, 1, 1), (1024, 1, 1), a),
            Launch("beams", "nk_assign_plan", (1, 1, 1), (1024, 1, 1), a),
            Launch("beams", "nk_assign_fill", (rows + -(-tokens // 256), 1, 1), (256, 1, 1), a)]


SELECT_SEG, SELECT_HEADS = 8192, 2048  # logits of a workgroup, lists of a group at most (beams.hip)


def select_segments(dtype, vocab) -> int:
    """Workgroups of a row, wherever it begins in its 16 bytes."""
    return -(-(vocab + 16 // dt.itemsize(dtype) - 1) // SELECT_SEG)


def select_workspace_bytes(dtype, groups, beams, vocab) -> int:
    return 8 * groups * beams * select_segments(dtype, vocab) * (1 + beams)


def beam_select(dtype, groups, beams, vocab, ld, end, *, x, scores, ended, tokens, parents, out, ends, ws) -> List[Launch]:
    """The beams of every group; ``ws``: ``select_workspace_bytes``."""
    nseg = select_segments(dtype, vocab)
    if not (groups >= 1 and 1 <= beams <= MAX_BEAMS and 1 <= vocab <= 2**22 and beams * nseg <= SELECT_HEADS):
        raise LaunchError(f"beam_select: {groups} groups of {beams} beams of {vocab}")
    n = groups * beams * nseg
    if n >= 2**31 or not ws or ws % 8:
        raise LaunchError("beam_select: too many rows for one launch, or no workspace")
    a = _fields(SelectArgs(), x=x, scores=scores, ended=ended, tokens=tokens, parents=parents, out=out, ends=ends, sums=ws,
                best=ws + 8 * n, ld=ld, groups=groups, beams=beams, vocab=vocab, nseg=nseg, end=end)
    return [Launch("beams", f"nk_select_top_{dtype_tag(dtype)}", (n, 1, 1), (256, 1, 1), a,
                   bytes=groups * beams * vocab * dt.itemsize(dtype)),
            Launch("beams", "nk_select_pick", (groups, 1, 1), (1024, 1, 1), a)]


def beam_reorder(groups, beams, width, page, pages, hkv, row, *, parents, lens, tables, k, v, ke=0, ve=0) -> Launch:
    """Tables, caches (rows of ``row`` bytes) and exponents updated in place."""
    unit = 16 if not any(p % 16 for p in (k, v, row)) else 1
    if not (groups >= 1 and 1 <= beams <= MAX_BEAMS and width >= 1 and pages >= 1 and page >= 1 and row >= 1
            and width * page < 2**30 and page * row // unit < 2**31):
        raise LaunchError(f"beam_reorder: {groups} groups of {beams} beams, pages of {page} rows")
    # (a page in part filled has a row less)
    a = _fields(ReorderArgs(), parents=parents, lens=lens, tables=tables, k=k, v=v, ke=ke, ve=ve, row=row, groups=groups,
                beams=beams, width=width, page=page, pages=pages, hkv=hkv, tblocks=-(-width // 256),
                kblocks=max(-(-(page - 1) * row // unit // 256), 1))
    n = groups * (a.tblocks + 2 * a.kblocks + (1 if ke else 0))
    if n >= 2**31:
        raise LaunchError("beam_reorder: too many workgroups for one launch")
    kk = next(c for c in (4, 8, MAX_BEAMS) if beams <= c)
    return Launch("beams", f"nk_beam_reorder{unit}_k{kk}", (n, 1, 1), (256, 1, 1), a)


# ---------------------------------------------------------------------------
# Patterns
# ---------------------------------------------------------------------------
class UpdateMatch(Match):
    """The nodes of one call: the parts that are read, by name.  ``views``:
    the operands that are read through strides."""

    name = "update"

    def __init__(self, nodes: List[Node], views: Dict[int, View] = {}):
        self.parts = {n.attrs["part"]: n for n in nodes}
        self.operands = nodes[0].inputs
        self.at = nodes[0].attrs
        targets = [n.attrs["target"] for n in nodes if "target" in n.attrs]
        self.updated = frozenset(self.operands[t].id for t in targets)
        inputs = [views[i].base if i in views else v for i, v in enumerate(self.operands)]
        super().__init__(nodes, list(dict.fromkeys(inputs)), [n.out for n in nodes])

    def begin(self, plan, results: Dict[str, int]) -> Tuple[list, dict]:
        """Steps that copy what is not updated in the caller's buffer, and
        where each part goes: its value, or space for a result (its bytes by
        name) that nobody reads."""
        steps, where = [], {}
        for part, n in self.parts.items():
            where[part] = n.out
            if "target" not in n.attrs:
                continue
            v = n.inputs[n.attrs["target"]]
            src, dst = plan.buffers[plan.slot(v).buffer], plan.buffers[plan.slot(n.out).buffer]
            own = src is dst or dst.kind == "output" and src.kind == "input" and plan.alias_outputs.get(dst.name) == src.name
            if not own:
                steps.append(G.ProgramStep(f"copy {v!r}", G.flat_copy_program(v), n.out))
        for part, nbytes in results.items():
            if part not in where:
                where[part] = Slot(plan.add_buffer(max(nbytes, 4), "temp", f"{self.name}.{part}"))
        return steps, where


class AssignMatch(UpdateMatch):
    name = "assign_pages"

    def steps(self, plan):
        tables, lens, news = self.operands
        rows, width = tables.shape
        at = self.at
        steps, to = self.begin(plan, {"starts": 4 * rows + 4, "slots": 4 * at["tokens"], "free": 4})
        ws = Slot(plan.add_buffer(assign_workspace_bytes(rows, width, at["pages"], at["tokens"]), "temp", "assign_pages.plan"))

        def make(addr):
            return assign_pages(rows, width, at["page"], at["pages"], at["tokens"], lens=addr(lens), news=addr(news), ws=addr(ws),
                                **{part: addr(v) for part, v in to.items()})

        desc = f"assign pages {at['tokens']} tokens of {rows} sequences, {at['pages']} pages of {at['page']}"
        return steps + [LaunchStep("assign_pages", desc, self.inputs, self.outputs, make)]


class SelectMatch(UpdateMatch):
    name = "beam_select"

    def __init__(self, nodes):
        self.x, st = _strided(nodes[0].inputs[0])
        self.ld = st[0]
        super().__init__(nodes, {0: self.x})

    def steps(self, plan):
        x, scores, ended = self.operands
        groups, beams = scores.shape
        size = 4 * groups * beams
        steps, to = self.begin(plan, {p: size for p in ("tokens", "parents", "scores", "ended")})
        ws = Slot(plan.add_buffer(select_workspace_bytes(x.dtype, groups, beams, x.shape[1]), "temp", "beam_select.segments"))

        def make(addr):
            return beam_select(x.dtype, groups, beams, x.shape[1], self.ld, self.at["end"], x=_at(addr, self.x),
                               scores=addr(scores), ended=addr(ended), tokens=addr(to["tokens"]), parents=addr(to["parents"]),
                               out=addr(to["scores"]), ends=addr(to["ended"]), ws=addr(ws))

        desc = f"beam select {groups}x{beams} of {x.shape[1]}"
        return steps + [LaunchStep("beam_select", desc, self.inputs, self.outputs, make)]


class ReorderMatch(UpdateMatch):
    name = "beam_reorder"

    def steps(self, plan):
        parents, lens, tables, key = self.operands[:4]
        pages, page, hkv, dim = key.shape
        groups, beams = parents.shape
        steps, to = self.begin(plan, {})

        def make(addr):
            names = {"tables": "tables", "key_cache": "k", "value_cache": "v", "key_exps": "ke", "value_exps": "ve"}
            return beam_reorder(groups, beams, tables.shape[1], page, pages, hkv, hkv * dim * dt.itemsize(key.dtype),
                                parents=addr(parents), lens=addr(lens), **{names[p]: addr(v) for p, v in to.items()})

        desc = f"beam reorder {groups}x{beams}, pages of {page}"
        return steps + [LaunchStep("beam_reorder", desc, self.inputs, self.outputs, make)]


def calls(L, kinds):
    """The live nodes of ``kinds``, those of one call together: they follow
    each other in the trace, over the same operands and with the same
    attributes (two such calls, of which one is read for what the other is
    not, are one)."""
    def call(n):
        return n.op, [v.id for v in n.inputs], {k: x for k, x in n.attrs.items() if k not in ("part", "target")}

    group: List[Node] = []
    for n in L.live + [None]:
        if group and (n is None or call(n) != call(group[0]) or any(m.attrs["part"] == n.attrs["part"] for m in group)):
            yield group
            group = []
        if n is not None and n.op in kinds:
            group.append(n)


class BeamPattern:
    KINDS = {"assign_pages": AssignMatch, "beam_select": SelectMatch, "beam_reorder": ReorderMatch}

    def find(self, L):
        for group in calls(L, self.KINDS):
            m = self.KINDS[group[0].op](group)
            if m.validate(L):
                yield m
