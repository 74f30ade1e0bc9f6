"""The rule that chooses a product's form, on 148 SMs."""

from __future__ import annotations

import random
import re
from pathlib import Path

import pytest

from quantem.cuda import _core

SMS = 148


def test_every_form_is_chosen_by_some_size_and_no_other():
    """Forms: few rows, a tile per CTA, a tile per pair of CTAs (256 columns)."""
    rng = random.Random(1)
    seen = set()
    for _ in range(20000):
        rows, n, k = (int(2 ** rng.uniform(0, top)) for top in (21, 13, 13))
        product, dtype = rng.randrange(4), rng.choice([_core.BF16, _core.E4M3])
        form, cols, parts, rounds = _core.linear_act_form(product, rows, n, k, dtype, SMS)
        assert parts >= 1 and rounds >= 1
        seen.add((form, cols))
        if form == 0:
            assert product == 0 and parts in (1, 2, 4, 8)
    assert seen == {(0, 16), (0, 32), (0, 64), (0, 128), (1, 64), (1, 128), (1, 256), (2, 256)}


@pytest.mark.parametrize("product,rows,n,k", [(4, 1, 1, 1), (-1, 1, 1, 1), (0, 0, 1, 1), (0, 1, 0, 1), (0, 1, 1, 0)])
def test_form_refuses(product, rows, n, k):
    with pytest.raises(RuntimeError):
        _core.linear_act_form(product, rows, n, k, _core.BF16, SMS)


def test_parts_of_the_weight_gradient():
    """At least 512 rows each, at most 32768."""
    assert _core.linear_act_form(3, 300, 64, 64, _core.BF16, SMS)[2] == 1
    assert _core.linear_act_form(3, 5000, 64, 64, _core.BF16, SMS)[2] == 9
    assert _core.linear_act_form(3, 200000, 64, 64, _core.BF16, SMS)[2] == 148
    assert _core.linear_act_form(3, 2**22, 4096, 4096, _core.BF16, SMS)[2] == 2**22 // 32768


def test_decoder_kernels_check_their_indexes_in_the_debug_build():
    """Every kernel that reads or writes global memory by itself goes through a
    check; kernels are found by their __global__."""
    csrc = Path(__file__).resolve().parents[1] / "quantem-cuda_b200" / "csrc"
    for name in ("rms_norm.cu", "linear_act.cu"):
        source = (csrc / name).read_text()
        parts = re.split(r"^__global__ ", source, flags=re.M)[1:]
        assert len(parts) >= 4
        for part in parts:
            body = part[: part.index("\n}\n")]
            if re.match(r".*\bzero_kernel\b", body, flags=re.S):
                continue  # its loop's condition is the bound
            through = r"QC_IN_BOUNDS|in_array|in_rows|at_inside|inside\(|FewEpilogue|span\."
            assert re.search(through, body), f"{name}: {body[:120]}"
