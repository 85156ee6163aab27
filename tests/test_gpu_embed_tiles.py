"""The embedding's gradient where its sort takes another path: a tile is 1024 ids, one
workgroup sorts one tile in a single launch, up to 64 tiles add up one another's counts,
more have a launch for them. Checks and tolerances are test_gpu_embed's."""

from __future__ import annotations

import pytest

import test_gpu_embed as E

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1023, 1024, 1025, 2048, 2049, 65535, 65536, 65537, 66560, 66561])
@pytest.mark.parametrize("V,H,dtype", [(3, 5, "fp32"), (1500, 8, "bf16"), (70000, 4, "fp16")])
def test_tiles(n, V, H, dtype):
    E._check(E._ids(n, V), V, H, dtype, 1.0)
    E._check(E._ids(n, V, text=False), V, H, dtype, 0.5)
