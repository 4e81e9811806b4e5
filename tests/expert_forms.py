"""Shapes that between them run every form of the expert products' kernels and of the routing, each with the form that
the library's rules (csrc/mx_rule.h) give it on 256 CUs."""
from collections import namedtuple

from tinyoai_amd import weights as W

PAIRS = [(W.MXFP4, W.F32), (W.MXFP4, W.F16), (W.MXFP4, W.BF16), (W.MXFP4, W.MXFP4), (W.BF16, W.F32), (W.BF16, W.F16),
         (W.BF16, W.BF16)]
PLANES = {W.F32: 3, W.F16: 2, W.BF16: 1, W.MXFP4: 0}
TAIL = 3  # rows behind the last group

Form = namedtuple("Form", "form fmt xdtype gate counts rows cols odtype")


def few_forms():
    """Few rows for each expert: a column tile and two; up to 24, 32 and more chunks of columns; some with several
    units of 16 rows (an odd number) for a block."""
    cols = {W.MXFP4: {3: (160, 768), 4: (3328, 4096), 16: (4224, 6912)}, W.BF16: {3: (72, 1536), 4: (1608, 2048), 16: (2056, 4096)}}
    for fmt, xd in PAIRS:
        for gate in (False, True):
            for chunks, lengths in cols[fmt].items():
                if chunks == 16 and gate and xd != W.MXFP4:
                    continue
                for tiles, counts in ((1, [1, 0, 0, 0, 0, 1, 0, 0, 0, 0]), (2, [3, 0, 17, 1, 0, 12, 2, 0])):
                    for i, k in enumerate(lengths):
                        form = ("few", 16, 1, 4) if chunks == 16 else ("few", 8, tiles, chunks)
                        yield Form(form, fmt, xd, gate, counts, (70, 2500)[i == 0], k, (W.F32, W.BF16)[i])


def tile_forms():
    """More rows: each tile, at one step of columns, fewer steps than the ring holds and more; rows and groups of no
    whole tile."""
    for fmt, xd in PAIRS:
        p = PLANES[xd]
        tiles = [(64, 256), (64, 128), (32, 128)]
        if fmt == W.BF16 or p == 0:
            tiles.insert(0, (128, 256))
        if fmt == W.BF16 and p == 1:
            tiles.insert(0, (256, 256))
        for bm, bn in tiles:
            counts = {256: [380, 421], 128: [150, 0, 133, 240], 64: [80, 70, 0, 160], 32: [80, 70, 0, 160]}[bm]
            stored = {(256, 256): 12180, (128, 256): 5940, (64, 256): 5940, (64, 128): 3850, (32, 128): 300}[bm, bn]
            for gate in (False, True):
                for i, k in enumerate((32, 160, 544) if fmt == W.MXFP4 else (40, 136, 515)):
                    yield Form(("tile", bm, bn, 0), fmt, xd, gate, counts, stored // 2 if gate else stored, k,
                               (W.F32, W.F16, W.BF16)[(i + gate) % 3])


def run_forms():
    """One group of long rows, whose sums go to totals: (form, fmt, x's type, rows of x, rows of the matrix, columns)."""
    cols = {0: 65664, 1: 16448, 2: 4160, 3: 2752}
    for fmt, xd in PAIRS:
        p = PLANES[xd]
        yield ("tile", 64, 256, 1), fmt, xd, 1024, 4096, cols[p]
        yield ("tile", 64, 128, 1), fmt, xd, 1024, 1664, cols[p]
        yield ("tile", 32, 128, 1), fmt, xd, 64, 64, cols[p] * (4 if p else 2)
        if fmt == W.BF16:
            yield ("tile", 128, 256, 1), fmt, xd, 2048, 3328, cols[p]


# (path, experts of a lane), tokens, experts, choices
ROUTES = [(("one_block", 1), 5, 40, 8), (("one_block", 2), 32, 100, 8), (("one_block", 4), 8, 200, 8),
          (("one_block", 8), 8, 512, 4), (("one_block", 16), 7, 1000, 32), (("by_expert", 1), 100, 64, 4),
          (("by_expert", 2), 1000, 128, 8), (("by_expert", 4), 33, 256, 8), (("by_expert", 8), 700, 300, 5),
          (("by_expert", 16), 40, 1024, 8), (("by_tokens", 1), 2500, 64, 4), (("by_tokens", 2), 1300, 128, 8),
          (("by_tokens", 2), 9000, 65, 1), (("by_tokens", 4), 4500, 256, 2), (("by_tokens", 8), 1100, 512, 8),
          (("by_tokens", 8), 8500, 300, 1), (("by_tokens", 16), 600, 700, 32)]
