"""The choice of the block-scaled GEMM's tile against the launches that it was
fitted to (profiles/gemm_f8_tiles.csv, gemm_f8_e4m3_tiles.csv; no GPU)."""

import csv
import re
from pathlib import Path

import numpy as np
import pytest

from tjkernels import _lib

ROOT = Path(__file__).resolve().parents[1]
# (table, output type, bytes of an output element, list of tiles, its slowdown: geometric mean and worst)
TABLES = [("gemm_f8_tiles", _lib.BF16, 2, "kPlans", 0.0045, 0.09), ("gemm_f8_e4m3_tiles", _lib.E4M3, 1, "kPlansF8", 0.0025, 0.075)]


def _table(name):
    """(tile sizes, [(m, n, k, GELU)], microseconds)"""
    rows = list(csv.reader(open(ROOT / "profiles" / f"{name}.csv")))
    assert rows[0][:4] == ["m", "n", "k", "epilogue"]
    sizes = [tuple(int(v) for v in re.match(r"(\d+)x(\d+)", h).groups()) for h in rows[0][4:]]
    assert {r[3] for r in rows[1:]} == {"bias", "gelu"}
    return sizes, [(*map(int, r[:3]), r[3] == "gelu") for r in rows[1:]], np.array([[float(v) for v in r[4:]] for r in rows[1:]])


@pytest.mark.parametrize("name,out,es,_list,mean,worst", TABLES)
def test_chosen_tiles_are_near_the_best(name, out, es, _list, mean, worst):
    _, shapes, us = _table(name)
    assert min(n for _, n, _, _ in shapes) == min(k for _, _, k, _ in shapes) == 128
    plans = [_lib.load().tjk_gemm_f8_default_plan(m, n, k, out, int(gelu)) for m, n, k, gelu in shapes]
    slower = us[np.arange(len(us)), plans] / us.min(axis=1)
    assert np.log(slower).mean() <= np.log1p(mean) and slower.max() <= 1 + worst


@pytest.mark.parametrize("name,out,es,plans,_mean,_worst", TABLES)
def test_estimates_are_the_fit_of_the_tables(name, out, es, plans, _mean, _worst):
    """Non-negative least squares of the relative error, weighted towards tiles
    near the best of their launch, gives the coefficients in the source (three
    decimals)."""
    nnls = pytest.importorskip("scipy.optimize").nnls
    sizes, shapes, us = _table(name)
    source = (ROOT / "tiktok-techjam-2026_amd" / "csrc" / "gemm_f8.hip").read_text()
    tiles = {t: [int(v) for v in g.split(",")[:5]]
             for g, t in re.findall(r"typedef F8Geom<([^>]*)> (\w+);", source)}
    entries = re.findall(r"\{(\w+)::BM, \1::BN, (\d), \1::KG, \{([^}]*)\}\}",
                         re.search(rf"{plans}\[\] = \{{(.*?)\}};", source, re.S)[1])
    assert len(entries) == len(sizes)
    best = us.min(axis=1)
    for (tile, per_cu, coef), (bm, bn), t in zip(entries, sizes, us.T):
        fm, fn, wm, wn, groups = tiles[tile]
        assert (32 * fm * wm, 32 * fn * wn) == (bm, bn)
        terms = []
        for m, n, k, gelu in shapes:
            count, steps = -(-m // bm) * -(-n // bn), -(-(-(-k // 128)) // groups)
            full, rest = divmod(count, 256 * int(per_cu))
            rounds, load = full + (rest > 0), full * int(per_cu) + -(-rest // 256)
            terms.append([1, rounds, rounds * steps, load, load * steps, m * n * es / 5e6, load * gelu])
        w = np.where(t < 1.3 * best, 3, np.where(t < 2 * best, 1, 0.25)) / t
        fitted, _ = nnls(np.array(terms, float) * w[:, None], t * w)
        assert np.abs(fitted - [float(c.strip(" f")) for c in coef.split(",")]).max() <= 6e-4, tile
