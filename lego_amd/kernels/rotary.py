"""Generator of the kernel that turns queries and keys by their positions.

A token's angles are shared by its heads, so a workgroup takes whole tokens: the units of work are those of a
``[tokens, heads, units of a head]`` box, row-major, a lane after the other.
"""
from __future__ import annotations

from ..lego import OrderBy, Row
from .common import BANNER, Emitted, code, idx, size, template, tidy

TOKENS = 1
THREADS = 256
MOST = 256      # elements of a head that are turned at most: the angles of a token are kept in LDS


def emit():
    heads, units, u = size("heads"), size("units"), idx("u")
    slot, head, unit = (tidy(e, {u: (0, TOKENS * heads * units)}) for e in OrderBy(Row(TOKENS, heads, units)).TileBy([TOKENS, heads, units]).inv(u))
    text = template("rotary.hip.j2").render(
        banner=BANNER, TOKENS=TOKENS, THREADS=THREADS, MOST=MOST, slot=code(slot), head=code(head), unit=code(unit),
        unit_layout=f"OrderBy(Row({TOKENS}, heads, units)).TileBy([{TOKENS}, heads, units]).inv(u)")
    return Emitted("rotary.hip", text, ["lego_rotary_launch"]), dict(MOST=MOST)
