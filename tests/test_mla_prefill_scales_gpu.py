"""GPU: chunk attention where the latent and the rope part of the queries differ by many powers of two
(both are scaled by one factor per row).  Tolerances as over short contexts."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_mla_prefill_gpu import Problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ctx", [200, 3000])
@pytest.mark.parametrize("latent,rope,k_rope", [(1e-30, 2e4, 2e4), (1e-36, 1.0, 1e6), (1e-18, 1e3, 1e3), (1e-7, 1.0, 1.0), (1e30, 1.0, 1.0),
                                                (0.0, 1e5, 1e5), (1e-30, 0.0, 1.0), (1.0, 1e-30, 1.0), (1.0, 1e20, 1e-19)])
def test_parts_of_very_different_sizes(latent, rope, k_rope, ctx):
    p = Problem([3, 1], [ctx, 77], 16, 64, True, seed=7)
    p.q[..., :512] *= latent
    p.q[..., 512:] *= rope
    p.rope *= k_rope
    p.scale = 1.0 / (24.0 * max(latent, rope * k_rope))
    out, lse = p.run()
    assert rt.device_errors() == 0
    p.check(out, lse)
