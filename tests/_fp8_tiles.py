"""Which tile an E4M3 product takes, by the costs in csrc/fp8_gemm.hip."""

import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mega-moe-td_amd", "csrc", "fp8_gemm.hip")


def costs(name):
    text = open(SOURCE).read()
    table = re.search(r"constexpr TileCost " + name + r"\[\] = \{(.*?)\};", text, re.S)[1]
    found = re.findall(r"\{(\d+), (\d+), (\d+), ([\d.e-]+), ([\d.e-]+), (true|false)\}", table)
    return [(int(bm), int(bn), int(step), float(tile), float(byte), several == "true")
            for bm, bn, step, tile, byte, several in found]


def ceil(n, d):
    return -(-n // d)


def tile(m, n, k, wide):
    """(rows, columns) of the tile of an m x n x k product; ``wide``: results in 32 bits."""
    assert m > 16 and k >= 128
    if wide and ceil(m, 128) * ceil(n, 128) >= 1024:
        return 128, 128
    times = []
    for bm, bn, step, fixed, byte, several in costs("kWideCosts" if wide else "kTileCosts"):
        tiles = ceil(m, bm) * ceil(n, bn)
        rounds = ceil(tiles, 256)
        if several and rounds > 1:
            rounds = max(rounds - 0.58, tiles / 256)
        if k >= step:
            times.append((rounds * (fixed + byte * k), bm, bn))
    return min(times)[1:]
