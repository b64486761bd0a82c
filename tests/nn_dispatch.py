"""Which kernels of the gated feed-forward block a call runs, by its sizes: the
launch rules of csrc/ffn.hpp restated, so that the tests can choose rows at the
edges of a launch's parts and show that their sizes reach every kernel.  The
sizes of the workspaces, which the library works out by the same rules without
a GPU, hold this file to them.
"""
from __future__ import annotations

CUS = 256
LDS_BYTES = 160 * 1024
DW_WAVES = 4
MADE = (1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16)


def ceil_div(a, b):
    return -(-a // b)


class Plan:
    """size: bytes of an element (4 or 2)."""

    def __init__(self, size, rows, dim, hidden):
        self.size, self.rows, self.dim, self.hidden = size, rows, dim, hidden
        self.e = 16 // size                       # elements of a piece
        self.ht = self.e // 4                     # 16-row tiles of a block
        self.kb = 4 * self.e                      # indices of a block
        n = ceil_div(dim, self.kb)
        self.dk = next(m for m in MADE if n <= m)
        self.tiny = dim < self.e
        self.f = self.dk * self.ht                # fragments
        self.hblocks = ceil_div(hidden, self.kb)

    def packed(self, mats):
        return self.hblocks * mats * self.f * 1024

    def few_limit(self):
        return CUS * (64 if self.f <= 4 else 32 if self.f <= 8 else 16)

    def tail(self, tiles, rows_of_workgroup=8):
        per_round = 16 * tiles * rows_of_workgroup * (2 if self.f <= 8 else 1) * CUS
        rest = self.rows % per_round
        return rest if self.rows > per_round and rest <= 16 * CUS else 0

    def few(self, name, rows):
        tiles = 1 if rows <= 16 * CUS else 2
        groups = ceil_div(rows, 16 * tiles)
        splits = max(1, min(CUS // groups, ceil_div(self.hblocks, 8))) if self.hblocks > 24 else 1
        out = [(name, self.dk, tiles, self.tiny)]
        return out + [("join", splits > 1)] if splits > 1 else out

    def forward(self):
        """The kernels of a forward call as (name, blocks of the width, row tiles a wave, narrow)."""
        pieces = self.hidden >= self.e
        if self.rows <= self.few_limit() and pieces:
            return self.few("fwd_few", self.rows)
        out = [("pack", False)]
        if self.f <= 4 and self.packed(3) <= LDS_BYTES:
            return out + [("fwd_all", self.dk, 1 if self.size == 4 else 2, self.tiny)]
        tiles = 1 if self.size == 4 or self.f <= 8 else 2
        tail = self.tail(tiles) if pieces else 0
        if tail:
            out += self.few("fwd_few", tail)
        main = self.rows - tail
        return out + [("fwd", self.dk, tiles if tiles == 2 and main >= 32 * 4 * CUS else 1, self.tiny)]

    def input_gradient(self):
        if self.rows <= self.few_limit():
            return self.few("dx_few", self.rows)
        if self.f <= 4 and self.packed(3) <= LDS_BYTES:
            return [("dx_all", self.dk, 1, self.tiny)]
        tiles = 2 if self.size == 2 and self.f == 8 else 1
        tail = self.tail(tiles)
        out = self.few("dx_few", tail) if tail else []
        main = self.rows - tail
        return out + [("dx", self.dk, tiles if tiles == 2 and main >= 32 * 4 * CUS else 1, self.tiny)]

    def occupancy(self, nh):
        n = self.dk * nh
        return 4 if n == 1 else 3 if n == 2 else 2 if n <= 5 else 1

    def weight_gradient(self):
        """(hidden tiles a wave, slices, groups, tiles, blocks of rows a group)."""
        tiles = self.hblocks * self.ht
        nh = (2 if self.size == 2 and self.dk <= 2 else 1) if tiles > DW_WAVES else 1
        slices = ceil_div(tiles, DW_WAVES * nh)
        blocks = ceil_div(self.rows, self.kb)
        most = max(1, 1024 // DW_WAVES * self.occupancy(nh) // slices)
        groups = min(most, max((blocks + 3) // 4, min(blocks, CUS // slices)))
        each = ceil_div(blocks, groups) if groups else 0
        groups = ceil_div(blocks, each) if each else 0
        return nh, slices, groups, slices * DW_WAVES * nh, each

    def backward(self):
        nh, slices, groups, _, each = self.weight_gradient()
        out = [("pack", True)] + self.input_gradient() + [("dw", self.dk, nh, self.tiny)]
        # a group of one block, of two and more: the double buffer's three states
        return out + [("dw_blocks", min(each, 3)), ("dw_groups", groups > 1)]

    def forward_workspace(self):
        return self.packed(3) + CUS * self.f * 1024

    def backward_workspace(self):
        _, _, groups, tiles, _ = self.weight_gradient()
        return self.packed(5) + CUS * self.f * 1024 + groups * tiles * 3 * self.f * 1024

    def edge_rows(self):
        """Rows on both sides of every group's and the last blocks' edges."""
        _, _, groups, _, each = self.weight_gradient()
        edges = {g * each * self.kb for g in range(groups)} | {self.rows}
        edges |= {self.rows // self.kb * self.kb, (self.rows // self.kb - 1) * self.kb, self.rows - self.kb, self.kb}
        rows = {r for e in edges for r in (e - 1, e)}
        return sorted(r for r in rows if 0 <= r < self.rows)


class NormPlan:
    """Layer norm's launch: lanes and pieces of a row, rows of a workgroup at
    once, workgroups of the forward and of the backward."""

    def __init__(self, size, rows, dim):
        pieces = ceil_div(dim, 16 // size)
        shapes = [(1 << i, 1) for i in range(7)] + [(64, 2), (64, 4), (256, 2), (256, 4), (256, 8)]
        self.lanes, self.pieces = next(s for s in shapes if pieces <= s[0] * s[1])
        self.at_once = 256 // self.lanes
        self.forward_groups = min(ceil_div(rows, self.at_once), 4096)
        self.backward_groups = min(ceil_div(rows, self.at_once), 1024)

    def backward_workspace(self, dim):
        return self.backward_groups * 2 * dim * 4
