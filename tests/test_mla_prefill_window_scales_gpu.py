"""GPU: windowed chunk attention where the latent and the rope part of the queries differ by many powers
of two, in both of its forms (few rows: both scaled by one factor per row; large calls: bf16 as they
are).  Tolerances as over short contexts."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_mla_prefill_window_gpu import Windowed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,H,window", [(3, 16, 150), (3, 64, 900), (150, 64, 300)])
@pytest.mark.parametrize("latent,rope,k_rope", [(1e-30, 2e4, 2e4), (1e-36, 1.0, 1e6), (1e-18, 1e3, 1e3), (1e-7, 1.0, 1.0), (1e30, 1.0, 1.0),
                                                (0.0, 1e5, 1e5), (1e-30, 0.0, 1.0), (1.0, 1e-30, 1.0), (1.0, 1e20, 1e-19)])
def test_parts_of_very_different_sizes(latent, rope, k_rope, n, H, window):
    p = Windowed([n, 1], [3000, 77], H, 64, True, window, 10, seed=7)
    p.q[..., :512] *= latent
    p.q[..., 512:] *= rope
    p.rope *= k_rope
    p.scale = 1.0 / (24.0 * max(latent, rope * k_rope))
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)
