"""Workspace sizes of the gated projection over the rows (no GPU)."""
from __future__ import annotations

import pytest

# 128 experts of 4096 x 1408, sizes that are no multiple of 8, experts whose weights are
# so few that FP32 goes back to the plain form behind a step of tiles, one expert.
LAYERS = [(128, 4096, 1408), (64, 57, 25), (8, 1001, 333), (3, 8, 8), (4, 136, 72), (1, 16, 130),
          (1, 2400, 4), (1, 1, 1), (1024, 64, 32)]


@pytest.mark.parametrize("dtype", [0, 2], ids=["fp32", "bf16"])
@pytest.mark.parametrize("layer", LAYERS, ids=str)
def test_a_workspace_serves_fewer_rows(rrlib, layer, dtype):
    lib, (e, k, n) = rrlib.lib(), layer
    steps = {m * e + d for m in (1, 2, 4, 8, 16, 32, 64, 256, 512, 768) for d in (-1, 0, 1)}
    rows = sorted({int(1.09 ** i) for i in range(160)} | steps | {65534, 65535, 65536})
    for size in (lib.rr_grouped_gated_gemm_workspace_size,
                 lib.rr_grouped_gated_gemm_backward_workspace_size):
        sizes = [size(r, e, k, n, dtype) for r in rows]
        assert sizes == sorted(sizes)
