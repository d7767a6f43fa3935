"""A beam search's step over an 8-bit paged cache, and the operands of a run."""

import numpy as np

from nkipy_amd.core import tensor_apis as T

import beams_plain as B
import fp8_plain as Q
import serving_plain as P

GROUPS, BEAMS, PAGES, PAGE, HEADS, KV, DIM, VOCAB, END = 3, 4, 60, 8, 4, 2, 64, 300, 7
ROWS = GROUPS * BEAMS
ARRAYS = ("kc", "vc", "ke", "ve", "tables")


def step(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens, new, logits, scores, ended):
    """One token for every beam: tables, append, attention, choice, reordering."""
    starts, slots, free = T.assign_pages(tables, lens, new, pages=PAGES, page_size=PAGE, tokens=ROWS)
    q = T.rotary_append_fp8(q, k, v, cos, sin, kc, vc, ke, ve, tables, lens)
    out = T.paged_attention_fp8(q, kc, vc, ke, ve, tables, lens)
    tokens, parents, scores, ended = T.beam_select(logits, scores, ended, end_token=END)
    T.beam_reorder(parents, tables, lens, kc, vc, ke, ve)
    return out, slots, free, tokens, parents, scores, ended


def begin(rng):
    """The caches and tables before the first token, and the rotary tables."""
    kc, ke = Q.random_cache(rng, PAGES, PAGE, KV, DIM)
    vc, ve = Q.random_cache(rng, PAGES, PAGE, KV, DIM)
    ang = rng.standard_normal((40, DIM // 2)).astype(np.float32)
    return dict(kc=kc, vc=vc, ke=ke, ve=ve, tables=np.full((ROWS, 5), -1, np.int32), cos=np.cos(ang), sin=np.sin(ang))


def token(rng, i, t, scores, ended):
    """What step i brings."""
    g = lambda *s: P.cast(rng.standard_normal(s), t)  # noqa: E731
    return dict(q=g(ROWS, HEADS, DIM), k=g(ROWS, KV, DIM), v=g(ROWS, KV, DIM), lens=np.full(ROWS, i + 1, np.int32),
                new=np.ones(ROWS, np.int32), logits=B.logits(rng, ROWS, VOCAB, t), scores=scores, ended=ended)
