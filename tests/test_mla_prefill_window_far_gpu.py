"""GPU: windowed chunk attention at the end of sequences of nearly 2^31 tokens, all but their first and last
pages given back, in both of its forms."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_mla_prefill_window_gpu import Windowed

pytestmark = pytest.mark.gpu
PAGE, MOST = 4096, 2 ** 31 - 1
LAST = MOST // PAGE             # pages of the longest sequence: 2^31 - 4,096 tokens


@pytest.mark.parametrize("n,H,window,sinks", [(3, 16, 600, 20), (1, 64, 130, 0), (150, 64, 300, 100), (257, 20, 5000, 3)])
@pytest.mark.parametrize("short", [0, 1, 63, 64, 255, 257])
def test_the_end_of_the_longest_sequences(n, H, window, sinks, short):
    """The last tokens of a sequence of two and a bit pages, put there."""
    ctx = 3 * PAGE - short
    p = Windowed([n], [ctx], H, PAGE, True, window, sinks, seed=short)
    far = torch.full((1, LAST + 1), _lib.PAGE_TRIMMED, dtype=torch.int32, device="cuda")
    far[0, 0] = p.tables[0, 0]
    far[0, LAST - 2: LAST] = p.tables[0, 1:].cuda()
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for length in [LAST * PAGE - short] + [MOST] * (short == 0):
        seq = torch.tensor([length], dtype=torch.int32, device="cuda")
        out, lse = rt.mla_prefill(p.q, p.pool, None, 512, 64, far, cu, seq, n, MOST, bmm1_scale=p.scale, rope_cache=p.rope,
                                  return_lse=True, window=window, sinks=sinks)
        # (a longer one ends at the bound, flagged)
        assert rt.device_errors() == (_lib.DEVERR_SEQ_LEN if length == MOST else 0)
        p.check(out, lse)
