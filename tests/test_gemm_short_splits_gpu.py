"""The library's own split-K over contractions that leave a split a single step, after a kernel that left other numbers in
the LDS."""
from __future__ import annotations

import pytest
import torch

from llm_training_amd.ops.native import lib
from test_gemm_short_contraction_gpu import right

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("K,split", [(128, 2), (192, 2), (256, 4), (256, 2), (512, 4)])
@pytest.mark.parametrize("streamk", [True, False])
def test_imported_split_of_every_candidate(K, split, streamk):
    """Every candidate of x @ w^T with an imported split: the "Custom_" ones drop a split into single steps."""
    torch.manual_seed(K)
    M, N = 256, 1024
    x, w = torch.randn(M, K, device=DEV).bfloat16(), torch.randn(N, K, device=DEV).bfloat16()
    big = torch.full((2048, 2048), 1e15, device=DEV).bfloat16()
    y = torch.empty(M, N, device=DEV).bfloat16()
    key = f"tn_{N}_{M}_{K}_ld{K}_{K}_{N}_bf16" + ("" if streamk else "_nosk")
    try:
        for rank in range(24):
            lib().gemm_lt_adopt(f"{key} {rank} 0 name gsu{split}\n")
            big @ big
            try:
                lib().gemm_lt(w, x, y, True, False, N, M, K, K, K, N, False, streamk)
                done = True
            except RuntimeError as e:  # (a solution without a split form)
                assert "isAlgoSupported" in str(e) or "initialize" in str(e), e
                done = False
            line, = (ln.split() for ln in lib().gemm_lt_export().splitlines() if ln.startswith(key + " "))
            if int(line[1]) != rank:  # (fewer candidates than that: the heuristic's choice ran)
                break
            custom = line[3].startswith("Custom_") and K < 128 * split
            assert not (custom and line[4] != "gsu0"), line
            assert done or not custom, line
            assert not done or right(y, x, w.t()), line
    finally:
        lib().gemm_lt_adopt(f"{key} 0 0 name gsu0\n")
