"""Generator of the attention kernels: forward, backward, and drafted tokens over a paged cache.

A tile is 64 rows (keys, or queries in the backward pass) of a head, as ``[row][16-byte chunk]`` in LDS with the chunk index
XOR-rotated by a key of the row.  The kernels read it in two ways, as it lies (16 consecutive rows, the same chunk of each) and
transposed (four consecutive rows, 64 bytes of each), and the key has to keep both free of bank conflicts: its upper part
goes with the row's lowest bits and sends the four rows of a transposing read to four different 64-byte quarters of the banks,
its lower part with the next bits, so that 16 consecutive rows have 16 different places.
"""
from __future__ import annotations

import re

import sympy as sp

from ..lego import BitXor, GenP, OrderBy, Row
from .common import BANNER, Emitted, code, idx, size, template, tidy
from .gemm import XCDS, lane_and_unit, xcd_remap

ELEMENTS = {"f16": "_Float16", "bf16": "__bf16"}
HEADS = (64, 96, 128)      # computed head elements: a head of another size takes the next one, with zeros
MAX_HEAD = HEADS[-1]
ROWS = 64
WAVES = 4
LAZY = 8
PSHIFT = {"f16": 8, "bf16": 0}      # P is held as 2^PSHIFT P in the backward pass
JOIN_ROWS, JOIN_MANY, JOIN_FEW = 8, 4096, 8      # rows of a workgroup that joins parts, from how many rows on; parts that the lanes of a row go through
ORDERED = 512      # blocks of rows that are put in order of their work with documents, at most
TREE_PIECE = 1024      # entries of a page table in LDS
TREE_LEAST = 2      # tiles of a run at least


def tile_layout(rows, chunks):
    """``row*chunks + (chunk ^ key(row))`` for rows of 8 or 16 chunks (128 or 256 bytes; the banks are 256 bytes wide)."""
    assert chunks in (8, 16)

    def key(row):
        first = 4 * (row % 4) if chunks == 16 else 4 * ((row // 2) % 2)
        return first + (row // 4) % 4

    def forward(rc):
        row, ch = rc
        return row * chunks + BitXor(sp.sympify(ch), sp.sympify(key(row)))

    def backward(flat):
        row, p = flat // chunks, flat % chunks
        return (row, BitXor(sp.sympify(p), sp.sympify(key(row))))

    return OrderBy(GenP((rows, chunks), forward, backward)).TileBy([rows, chunks])


def _tile_params(head, waves):
    pitch = 64 if head <= 64 else 128
    chunks = pitch // 8
    lds = tile_layout(ROWS, chunks)
    l32, lhi, l16, lgrp, lane, wave = (idx(n) for n in ("l32", "lhi", "l16", "lgrp", "lane", "wave"))
    blk, ks, st, j, db, it = (idx(n) for n in ("blk", "ks", "st", "j", "db", "it"))
    rng = {l32: (0, 32), lhi: (0, 2), l16: (0, 16), lgrp: (0, 4), lane: (0, 64), wave: (0, waves), blk: (0, 2), ks: (0, head // 16),
           st: (0, 4), j: (0, 2), db: (0, head // 32)}
    # rows as they lie: row l32 of block blk, chunk 2 ks + lhi
    row_lane, row_units = lane_and_unit(16 * lds[32 * blk + l32, 2 * ks + lhi], (blk, ks), [(x, y) for x in range(2) for y in range(head // 16)],
                                        (l32, lhi), [(x, y) for x in range(32) for y in range(2)], 32 * pitch * 2)
    assert all(unit == (x * 32 * pitch * 2, 32 * y) for (x, y), unit in row_units.items())
    # transposed: source lane s of a group of 16 supplies row s/4 of four and 4 elements from 4 (s % 4) on of the group's 16
    tr_row = 16 * st + 8 * j + 4 * lhi + l16 // 4
    tr_chunk = 4 * db + 2 * (lgrp % 2) + (l16 % 4) // 2
    tr_lane, tr_units = lane_and_unit(16 * lds[tr_row, tr_chunk], (st, j, db), [(x, y, z) for x in range(4) for y in range(2) for z in range(head // 32)],
                                      (l16, lgrp, lhi), [(x, 2 * z + y, z) for x in range(16) for y in range(2) for z in range(2)], 8 * pitch * 2)
    assert all(unit == (x * 16 * pitch * 2 + y * 8 * pitch * 2, (32 * y) ^ (64 * z)) for (x, y, z), unit in tr_units.items())
    # memory -> LDS: copy `it` of wave w fills slots 64 (waves it + w) .. + 63; a lane's chunk is the same for all copies, its rows are a
    # whole number of rows apart
    g = idx("g")      # number of a copy among all waves'
    slot = 64 * (waves * it + wave) + lane
    copies = ROWS * pitch * 2 // 1024 // waves
    row_e, chunk_e = (tidy(e, {lane: (0, 64), wave: (0, waves), it: (0, copies)}) for e in lds.inv(slot))
    f_row, f_chunk = (sp.lambdify((it, wave, lane), e, [{"BitXor": lambda a, b: int(a) ^ int(b)}, "math"]) for e in (row_e, chunk_e))
    for w in range(waves):
        for x in range(64):
            for c in range(copies):
                assert int(f_row(c, w, x)) == int(f_row(0, w, x)) + c * (ROWS // copies) and int(f_chunk(c, w, x)) == int(f_chunk(0, w, x))
    return dict(DC=head, PITCH=pitch, WAVES=waves, LAZY=LAZY, XCDS=XCDS,
                lds_layout=f"OrderBy(GenP(({ROWS}, {chunks}), row*{chunks} + (chunk ^ key(row)))).TileBy([{ROWS}, {chunks}])",
                row_lane=code(tidy(row_lane / 16, rng)), tr_lane=code(tidy(tr_lane / 16, rng)),
                any_row=code(tidy(lds.inv(64 * g + lane)[0], {lane: (0, 64), g: (0, ROWS * pitch // 512)})),
                any_chunk=code(tidy(lds.inv(64 * g + lane)[1], {lane: (0, 64), g: (0, ROWS * pitch // 512)})),
                fill_row=code(tidy(row_e.subs(it, 0), rng)), fill_chunk=code(tidy(chunk_e.subs(it, 0), rng)))


def emit():
    """The translation units: one per kernel, element type and computed head size."""
    units = []
    # workgroups one after the other have the same block of rows of different heads, the block with the most work first; heads whose number a multiple of XCDS allows it
    # stay on one XCD, neighbours together
    per, turn = size("per_xcd"), idx("turn")
    place = code(tidy(xcd_remap(per, turn), {turn: (0, XCDS * per)}))
    launch = f"Row(blocks, heads).inv(wg) = block, turn; head = OrderBy(Col(per_xcd, {XCDS})).TileBy([per_xcd, {XCDS}])[Row(per_xcd, {XCDS}).inv(turn)]"
    for dt, elt in ELEMENTS.items():
        for head in HEADS:
            params = dict(_tile_params(head, WAVES), banner=BANNER, elt=elt, dt=dt, tag=f"{dt}_d{head}", place=place, launch_layout=launch,
                          PSHIFT=PSHIFT[dt], RING=3 if head == 128 else 4)
            params |= dict(LEAST=TREE_LEAST, JOIN_ROWS=JOIN_ROWS, JOIN_MANY=JOIN_MANY, JOIN_FEW=JOIN_FEW, PIECE=TREE_PIECE)
            units.append(Emitted(f"tree_attention_{dt}_d{head}.hip", template("tree_attention.hip.j2").render(**params), [f"lego_tree_{dt}_d{head}_launch"]))
            for way in ("fwd", "bwd"):
                name = f"attention_{way}_{dt}_d{head}"
                units.append(Emitted(f"{name}.hip", template(f"attention_{way}.hip.j2").render(**params), [f"lego_{name}_launch"]))
    B, H, T = size("B"), size("H"), size("T")
    b, h, i = idx("b"), idx("h"), idx("i")
    stat = code(tidy(OrderBy(Row(B, H, T)).TileBy([B, H, T])[b, h, i], {b: (0, B), h: (0, H), i: (0, T)}))
    for name, text in (("b", "(size_t)b"), ("H", "a.heads"), ("T", "a.queries")):
        stat = re.sub(rf"\b{name}\b", text, stat)
    units.append(Emitted("attention_rows.hip", template("attention_rows.hip.j2").render(
        banner=BANNER, stat=stat, ORDERED=ORDERED, ORDER_FIGURES="forward 98 -> 84 us, dk and dv 191 -> 167, dq 146 -> 129 at 6 a launch", PSHIFT=PSHIFT["f16"], stat_layout="OrderBy(Row(batch, heads, queries)).TileBy([batch, heads, queries])[b, h, i]",
        parts_layout="OrderBy(Row(parts, 2, batch, key heads, keys, head))"),
        ["lego_attention_tiles_launch", "lego_attention_order_launch", "lego_attention_delta_launch", "lego_attention_join_launch"]))
    return units, dict(HEADS=HEADS, ORDERED=ORDERED, TREE_LEAST=TREE_LEAST, MAX_HEAD=MAX_HEAD, ELEMENTS=tuple(ELEMENTS))
