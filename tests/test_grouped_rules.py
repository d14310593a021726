"""The rule that decides between few rows and pairs (``csrc/mmoe_grouped_few.cu``), asked on the host.  No GPU involved."""

import os
import shutil
import subprocess

import pytest

import grouped_shapes as S
from helpers import ROOT


@pytest.fixture(scope="module")
def few(tmp_path_factory):
    """``few([(type, kind, rows, experts, channels, width), ...])`` -> whether the kernel for few rows takes each."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc is not installed")
    exe = str(tmp_path_factory.mktemp("rules") / "grouped_rules")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-o", exe, os.path.join(ROOT, "tests", "grouped_rules.cu")],
                   check=True, capture_output=True)

    def ask(products):
        text = "".join(f"{S.SMS} " + " ".join(map(str, p)) + "\n" for p in products)
        answers = subprocess.run([exe], input=text, check=True, capture_output=True, text=True).stdout.split()
        assert len(answers) == len(products)
        return [a == "1" for a in answers]

    return ask


def test_shapes_that_are_there_for_the_pairs(few):
    products = list(S.products())
    for product, is_few in zip(products, few(products)):
        assert not is_few, product


def test_either_side(few):
    """16 bits: two tiles to an SM up to 64 rows, two to three SMs above.  8 bits: up to 128 rows, and up to 64 rows an expert where its tiles fit or cost less."""
    cases = {
        (S.BF16, S.LINEAR, 64, 1, 5120, 5120): True, (S.BF16, S.LINEAR, 128, 1, 5120, 5120): True, (S.BF16, S.LINEAR, 192, 1, 5120, 5120): False,
        (S.BF16, S.GATED, 160, 1, 2304, 5120): False, (S.BF16, S.GATED, 6, 48, 2304, 5120): True, (S.BF16, S.GATED, 64, 8, 2304, 5120): True,
        (S.BF16, S.LINEAR, 64, 8, 5120, 2304): False, (S.BF16, S.LINEAR, 384, 48, 5120, 2304): False,
        (S.E4M3, S.LINEAR, 128, 1, 5120, 5120): True, (S.E4M3, S.LINEAR, 129, 1, 5120, 5120): False, (S.E4M3, S.GATED, 384, 48, 2304, 5120): True,
        (S.E4M3, S.GATED, 5000, 48, 2304, 5120): False, (S.E4M3, S.LINEAR, 512, 128, 2048, 768): False, (S.E4M3, S.GATED, 4096, 128, 768, 2048): True,
        (S.E4M3, S.LINEAR, 2304, 48, 5120, 2304): True, (S.E4M3, S.LINEAR, 3200, 48, 5120, 2304): False,
    }
    for (product, want), got in zip(cases.items(), few(list(cases))):
        assert got is want, product
