"""Every form that the 8-bit product takes has a case that the GPU tests hold to 64 bits.
Which form a size takes is asked of the plan itself, compiled for the host: the tile shape,
gated or not, either result, its tiles whole, in pieces or in pieces behind rounds of whole
ones, and a reduction that the tile's room for scales holds at once or not; of few tokens
the blocks of a workgroup and the types. A change of the plan's constants that leaves a
form without a case fails here."""

from __future__ import annotations

import random
import subprocess

import pytest

import test_gpu_fp8
import test_gpu_fp8_forms
import test_gpu_fp8_tiles
from h3_flash_amd._build import CSRC_DIR, HIPCC_FLAGS, INCLUDE_DIR, hipcc

PLAN = r"""
#include <cstdio>
#include "gemm_fp8_tile.h"
#include "linear_fp8.hip"

static int held_steps;  // K steps whose scales a tile holds at once

namespace h3a {
template <int TF, int NT, int SW, int SX>
hipError_t launch_linear_fp8_tile(const LinearFp8Params&, hipStream_t) {
    using T = Fp8Tile<TF, NT, SW, SX>;
    held_steps = kSegSteps * (T::kScaleRegs ? kHeldSegs : T::kSegs);
    return hipSuccess;
}
hipError_t launch_quantize(const QuantizeParams&, hipStream_t) { return hipSuccess; }
int64_t quantize_max_groups(bool) { return 1 << 30; }
}  // namespace h3a

int main() {
    int m, k, n, gated, x8, y8;
    uint8_t byte = 0;
    while (scanf("%d %d %d %d %d %d", &m, &k, &n, &gated, &x8, &y8) == 6) {
        h3a::LinearFp8Params p{};
        p.m = m; p.k = k; p.n = n; p.gated = gated;
        p.x_scale = x8 ? &byte : nullptr;
        p.y_scale = y8 ? &byte : nullptr;
        int64_t required, workspace;
        h3a::plan_linear_fp8(p, 256, &required, &workspace);
        if (p.shape == h3a::kRowsForm) {
            printf("0 %d %d\n", h3a::rows_form(p, 256).na, p.m <= 16 ? 1 : 2);
            continue;
        }
        if (p.shape < 0) return 1;
        const h3a::Shape& s = h3a::kShapes[p.shape];
        (void)s.launch(p, nullptr);
        printf("1 %d %d %d %d %d %d\n", s.tf, 16 * s.nt, p.split, p.n_full, p.m_tiles * p.n_tiles, held_steps);
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def form_of(tmp_path_factory):
    """A function: the forms of a list of (m, k, n, gated, x in 8 bits, result in 8 bits)."""
    try:
        compiler = hipcc()
    except RuntimeError:
        pytest.skip("hipcc not found")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.hip").write_text(PLAN)
    flags = [f for f in HIPCC_FLAGS if f != "-shared"]
    subprocess.run([compiler, *flags, "-O1", f"-I{INCLUDE_DIR}", f"-I{CSRC_DIR}", str(d / "plan.hip"), "-o", str(d / "plan")], check=True,
                   capture_output=True)

    def forms(sizes):
        text = "\n".join(" ".join(str(int(v)) for v in s) for s in sizes)
        out = subprocess.run([str(d / "plan")], input=text, check=True, capture_output=True, text=True).stdout.splitlines()
        assert len(out) == len(sizes)
        return [_form(s, *map(int, line.split())) for s, line in zip(sizes, out)]

    return forms


def _form(size, tiles, *plan):
    _, k, _, gated, x8, y8 = size
    common = ("gated" if gated else "plain", "to 8 bits" if y8 else "to bf16")
    if not tiles:
        blocks, token_blocks = plan
        return (f"{blocks} x {token_blocks} blocks", *common, "from 8 bits" if x8 else "from bf16")
    rows, tokens, split, whole, n, held = plan
    reduction = "whole" if whole == n else "pieces" if whole == 0 else "rounds, then pieces"
    steps = (k + 127) // 128
    longest = steps if whole else -(-steps // split)
    return (f"{rows} x {tokens} tiles", *common, reduction, "scales in turn" if longest > held else "scales at once")


def _cases():
    """The sizes that the GPU tests compare with 64 bits."""
    sizes = [(m, k, n, gated, x == "fp8", out == "fp8") for m, k, n, x, _, gated, _, _, _, out in test_gpu_fp8.CASES]
    for cases in (test_gpu_fp8_tiles.CASES, test_gpu_fp8_forms.CASES):
        sizes += [(m, k, n, gated, True, quantize) for m, k, n, gated, quantize in cases]
    return sizes + [(m, k, n, gated, x == "fp8", quantize) for m, k, n, gated, x, quantize in test_gpu_fp8_forms.FEW_TOKENS]


def test_every_form_has_a_case(form_of):
    covered = set(form_of(_cases()))
    rng = random.Random(7)

    def log_int(lo, hi):
        return round(lo * (hi / lo) ** rng.random())

    sizes = []
    for _ in range(400_000):
        gated, x8, y8 = (rng.random() < 0.5 for _ in range(3))
        m = log_int(1, 32) if rng.random() < 0.1 else log_int(17, 12480)
        sizes.append((m, 16 * log_int(1, 1400), (16 if y8 else 8) * log_int(1, 1800), gated, x8, y8))
    found = {}
    for size, form in zip(sizes, form_of(sizes)):
        if form not in found or size[0] * size[1] * size[2] < found[form][0] * found[form][1] * found[form][2]:
            found[form] = size
    assert len(found) > 80
    missing = {f: s for f, s in sorted(found.items()) if f not in covered}
    assert not missing, missing


def test_the_cases_of_a_form_take_it(form_of):
    # each of the cases that were added for one form still takes it, and no two the same
    for cases, sizes in ((test_gpu_fp8_forms.CASES, [(m, k, n, g, True, q) for m, k, n, g, q in test_gpu_fp8_forms.CASES]),
                         (test_gpu_fp8_forms.FEW_TOKENS, [(m, k, n, g, x == "fp8", q) for m, k, n, g, x, q in test_gpu_fp8_forms.FEW_TOKENS])):
        forms = form_of(sizes)
        assert len(set(forms)) == len(cases)
