"""Fits the prices of the block-scaled FP8 product's plans (vllm_amd/csrc/fp8_block_mm.hip) to their cold times, and says how good the plans are that they choose.

    python profiles/plan_prices/fp8_block.py [--fit]

Without --fit: the constants of the source, read from it.  With it: constants fitted to fp8_block_fit.csv.gz, from those of the source on.  Either is judged on
fp8_block.csv.gz, which the fit does not see (three sizes were drawn into both).  Lines: m,k,n,plan,us, a plan r<m-blocks>.<n-tiles>.<steps ahead>.<wavefronts> or
t<shape>.  Not every plan was timed for every size: plans for few rows where there are at most eight blocks of rows and all 16-row parts of the first hold rows; 64 x 64 and 64 x 128 tiles from 9 rows on, the
others from a quarter of their rows on (128: from 33 rows, 256: from 65).
"""
from __future__ import annotations

import gzip
import re
import sys
from collections import defaultdict
from pathlib import Path

import numpy as np

HERE = Path(__file__).resolve().parent
SOURCE = HERE.parent.parent / "vllm_amd" / "csrc" / "fp8_block_mm.hip"
CUS, SHAPES = 256, [(64, 64), (64, 128), (128, 128), (128, 256), (256, 128), (256, 256), (128, 64)]


def tables() -> tuple[dict, list]:
    """The constants of the source: by (steps ahead, wavefronts), by tile shape."""
    text = re.sub(r"//.*", "", SOURCE.read_text())

    def rows(name):
        body = re.search(name + r"\[[^=]*=\s*\{(.*?)\};", text, re.S).group(1)
        return [[float(x) for x in re.findall(r"-?\d+\.?\d*(?:e-?\d+)?", r)] for r in re.findall(r"\{([^{}]*)\}", body)]
    few, tiles = rows("ROWS_PRICE"), rows("TILE_PRICE")
    return {(1, 4): few[0], (1, 8): few[1], (2, 4): few[2], (2, 8): few[3]}, tiles


def cubes(*x):
    return np.cbrt(sum(v ** 3 for v in x))


def lds_bytes(k, mb, j, ahead, waves):
    steps = -(-(-(-k // 256)) // waves)
    return waves * ((mb + ahead * j) * 4096 + 4 * ((steps * 2 * mb * 16 + 63) // 64 * 64 + (steps * 2 + 63) // 64 * 64))


def rows_us(c, m, k, n, mb, j, ahead, waves):
    blocks = np.ceil(m / 16 / mb)
    per_cu = np.ceil(np.ceil(n / 16 / j) * blocks / CUS)
    slots = np.minimum(np.floor(160 * 1024 / lds_bytes(k.astype(int), mb, j, ahead, waves)), 16 // waves)
    side, rounds = np.minimum(per_cu, slots) * waves / 4, np.maximum(per_cu / slots, 1)
    step = cubes(c[0], c[1] * side * (mb + j), c[2] * side * mb * j)
    core = rounds * (c[3] + np.ceil(np.ceil(k / 256) / waves) * step + c[4] * mb * j * waves / 4)
    return c[7] + cubes(core, c[5] * 1e-6 * k * n * (1 + c[6] * (blocks - 1))) + c[8] * 1e-6 * m * n


def tile_us(c, m, k, n, shape):
    down, across = np.ceil(m / SHAPES[shape][0]), np.ceil(n / SHAPES[shape][1])
    full, rest = np.floor(down * across / CUS), (down * across) % CUS / CUS
    rounds = full + np.where(rest > 0, c[0] + (1 - c[0]) * rest, 0)
    core = rounds * (c[1] + np.ceil(k / 128) * c[2] * (1 + c[7] / down))
    return c[5] + cubes(core, c[3] * 1e-6 * k * n * (1 + c[4] * (down - 1))) + c[6] * 1e-6 * m * n


def price(plan, few, tiles, m, k, n):
    if plan[0] == "t":
        return tile_us(tiles[int(plan[1:])], m, k, n, int(plan[1:]))
    mb, j, ahead, waves = map(int, plan[1:].split("."))
    return rows_us(few[ahead, waves], m, k, n, mb, j, ahead, waves)


def load(path=HERE / "fp8_block.csv.gz"):
    """{plan: (m, k, n, us)} and [{plan: us}] by problem"""
    by_plan, by_problem = defaultdict(list), defaultdict(dict)
    with gzip.open(path, "rt") as f:
        for line in f:
            if not line.startswith("#"):
                m, k, n, plan, us = line.split(",")
                by_plan[plan].append((int(m), int(k), int(n), float(us)))
                by_problem[int(m), int(k), int(n)][plan] = float(us)
    return {p: np.array(v, dtype=float).T for p, v in by_plan.items()}, by_problem


def choice(by_problem, few, tiles):
    """Time of the cheapest plan over that of the fastest, for every problem."""
    out = []
    for (m, k, n), times in by_problem.items():
        args = [np.array([float(x)]) for x in (m, k, n)]
        out.append(times[min(times, key=lambda p: float(price(p, few, tiles, *args)[0]))] / min(times.values()))
    return np.array(out)


def fit(by_plan, few, tiles):
    from scipy.optimize import least_squares

    def solve(start, plans, at):
        def off(c):
            return np.concatenate([np.log(at(np.abs(c), p) / by_plan[p][3]) for p in plans])
        return np.abs(least_squares(off, start, loss="soft_l1", f_scale=0.05, max_nfev=100).x)
    for kind in few:
        plans = [p for p in by_plan if p[0] == "r" and p.endswith(".%d.%d" % kind)]
        few[kind] = solve(few[kind], plans, lambda c, p: price(p, {kind: c}, None, *by_plan[p][:3]))
    for shape in range(len(SHAPES)):
        if f"t{shape}" in by_plan:
            tiles[shape] = solve(tiles[shape], [f"t{shape}"], lambda c, p: tile_us(c, *by_plan[p][:3], shape))


if __name__ == "__main__":
    by_problem = load()[1]
    few, tiles = tables()
    if "--fit" in sys.argv:
        fit(load(HERE / "fp8_block_fit.csv.gz")[0], few, tiles)
        for name, rows in (("ROWS_PRICE", few.values()), ("TILE_PRICE", tiles)):
            print(name)
            for r in rows:
                print("    {" + ", ".join(f"{x:.4g}" for x in r) + "},")
    c = choice(by_problem, few, tiles)
    print(f"{len(c)} problems: the cheapest plan takes {c.mean():.4f} of the fastest one's time in the mean, 95 of 100 within {np.quantile(c, 0.95):.3f}")
