"""Windows, sinks and axes are whole numbers: what is not is refused, not cut off (a window of half a token
would be none at all)."""
import numpy as np
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt


@pytest.mark.parametrize("window,sinks", [(0.5, 0), (4.5, 0), (8, 0.25), (-0.5, 0), (float("nan"), 0), ("8", 0), (np.float32(0.5), 0),
                                          (8, torch.tensor(1.5)), (float("inf"), 0)])
def test_windows_that_are_not_whole(window, sinks):
    with pytest.raises((TypeError, ValueError, OverflowError)):
        rt._window(window, sinks)


@pytest.mark.parametrize("window,sinks", [(-1, 0), (4, -1), (0, 3)])
def test_windows_out_of_range(window, sinks):
    with pytest.raises(ValueError, match="window and sinks"):
        rt._window(window, sinks)


def test_whole_numbers_of_any_type():
    most = 2 ** 31 - 1
    for window, sinks, want in ((0, 0, (0, 0)), (1, 0, (1, 0)), (128.0, 4, (128, 4)), (np.int64(7), np.float32(3), (7, 3)), (True, False, (1, 0)),
                                (1 << 40, 1 << 40, (most, most)), (torch.tensor(9), torch.tensor(2), (9, 2))):
        got = rt._window(window, sinks)
        assert got == want and all(type(n) is int for n in got)


@pytest.mark.parametrize("axes", [(0, 0.5, 1, 1), [0, 1, 1.5, 0], (0, "1", 1, 1)])
def test_axes_that_are_not_whole(axes):
    for _ in range(2):
        with pytest.raises(TypeError, match="axes must be whole numbers"):
            rt._axes(axes, 2, 8)
    assert list(rt._axes([0, 1.0, np.int64(1), 0], 2, 8)) == [0, 1, 1, 0]


def test_sections_that_are_not_whole():
    for dealt in (False, True):
        with pytest.raises(TypeError, match="sections must be whole numbers"):
            rt.rope_axes((2.5, 1.5), 6, dealt=dealt)
    assert rt.rope_axes((2.0, 1), 6) == (0, 0, 1)


@pytest.mark.gpu
def test_the_entries_refuse_them():
    from test_mla_prefill_gpu import Problem

    p = Problem([1], [20], 4, 16, True)
    for kw in (dict(window=0.5), dict(window=4, sinks=0.5), dict(sinks=0.5)):
        with pytest.raises(TypeError, match="whole"):
            p.run(**kw)
    a, b = p.run(window=7, sinks=2), p.run(window=7.0, sinks=np.int64(2))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    for kw in (dict(window=0.5), dict(window=4, sinks=0.5)):
        with pytest.raises(TypeError, match="whole"):
            rt.trim_pages(i(-1, -1).view(1, 2), i(0), i(0), i(0, 0), 16, **kw)
    x, cos_sin = torch.randn(3, 8, device="cuda"), rt.rope_cos_sin(16, 8).cuda()
    with pytest.raises(TypeError, match="whole"):
        rt.apply_rope(x, torch.zeros(2, 3, dtype=torch.int64, device="cuda"), cos_sin, axes=(0, 0.5, 1, 1))
    assert rt.device_errors() == 0
