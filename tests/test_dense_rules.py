"""The rule for the tiles of dense products on CTA pairs (``csrc/mmoe_dense_rules.h``), compiled for the host.  No GPU involved."""

import os
import shutil
import subprocess

import pytest

import dense_widths as W
from helpers import ROOT

BF16, INT8 = 0, 2
LINEAR, GATED, GATED_GRAD = 0, 1, 2
WIDTHS = (128, 160, 192, 224, 256)


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    """``launches([[(type, kind, m, n, k, A transposed, B transposed), ...], ...])`` -> per launch ``([(columns, tiles), ...], stages)``."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc is not installed")
    exe = str(tmp_path_factory.mktemp("rules") / "dense_rules")
    subprocess.run([nvcc, "-std=c++17", "-Wno-deprecated-gpu-targets", "-o", exe, os.path.join(ROOT, "tests", "dense_rules.cpp")],
                   check=True, capture_output=True)

    def ask(products):
        text = "".join(f"{W.PAIRS} {len(ps)} " + " ".join(str(int(v)) for p in ps for v in p) + "\n" for ps in products)
        rows = [[int(v) for v in line.split()] for line in
                subprocess.run([exe], input=text, check=True, capture_output=True, text=True).stdout.splitlines()]
        assert len(rows) == len(products)
        return [([tuple(r[2 * i:2 * i + 2]) for i in range(len(r) // 2)], r[-1]) for r in rows]

    return ask


def _gated(t, m, n, k):
    return [(t, GATED, m, n, k, 0, 0)]


def _linear(t, m, n, k):
    return [(t, LINEAR, m, n, k, 0, 0)]


def test_the_tables_of_widths(launches):
    """Each shape takes the width that it is there for, and every one of the four launches of one product every width, in one turn of the pairs
    and in more, with a remainder of rows, of columns and of K."""
    seen = {}

    def note(name, product, shape):
        (cols, tiles), = product
        _, n, k, depth = shape
        width = cols // 2 if "gated" in name else cols
        if shape[0] % 256 and n % width and k % depth:
            seen.setdefault(name, set()).add((cols, tiles > W.PAIRS))

    for (m, h, i), want in W.BLOCKS.items():
        first, second, back, last = launches([
            _gated(BF16, m, i, h), _linear(BF16, m, h, i), [(BF16, GATED_GRAD, m, i, h, 0, 1), (BF16, LINEAR, h, i, m, 1, 1)],
            [(BF16, LINEAR, m, h, 2 * i, 0, 1), (BF16, LINEAR, 2 * i, h, m, 1, 1)]])
        got = (first[0][0][0], second[0][0][0], tuple(c for c, _ in back[0]), tuple(c for c, _ in last[0]))
        assert got == want, (m, h, i)
        note("gated", first[0], (m, i, h, 64))
        note("second", second[0], (m, h, i, 64))
    for name, table, product in (("gated, 8 bits", W.GATED, _gated), ("projection, 8 bits", W.PROJECTIONS, _linear)):
        for (m, n, k), want in table.items():
            (tiles, _), = launches([product(INT8, m, n, k)])
            assert tiles[0][0] == want, (name, m, n, k)
            note(name, tiles, (m, n, k, 128))
    for name, widths in seen.items():
        assert {(w, more) for w in WIDTHS for more in (False, True)} <= widths, (name, sorted(widths))
    assert len(seen) == 4
