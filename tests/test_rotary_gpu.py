"""GPU: rotary positions (apply_rope) and the rotated rope rows (write_nvfp4_rope_rotated) against
the rotation in 64 bits.

Tolerance per element: one rounding to the output type (2^-8, 2^-11, 2^-24 relative) and four
fp32 roundings of the two products, 4 * 2^-24 (|a c| + |b s|); 2^-25 for fp16 subnormals."""
import math

import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rotated(x, pos, cs, off, interleaved, inverse):
    """(y, |a c| + |b s| of each output) in float64; x [T, H, D]."""
    r = cs.shape[1]
    t = cs.double()[pos.long()][:, None]
    c, s = t[..., : r // 2], t[..., r // 2:] * (-1 if inverse else 1)
    i = torch.arange(r // 2, device=x.device)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    a, b = y[..., off + ia].clone(), y[..., off + ib].clone()
    y[..., off + ia], y[..., off + ib] = a * c - b * s, b * c + a * s
    size[..., off + ia], size[..., off + ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def check(got, want, size, dtype):
    tol = UNIT[dtype] * want.abs() + 4 * 2.0 ** -24 * size + 2.0 ** -25
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,H,D,r,off", [(1, 1, 64, 64, 0), (5, 3, 576, 64, 512), (17, 64, 128, 32, 0),
                                         (3, 2, 130, 34, 5), (2, 7, 100, 2, 98), (33, 5, 192, 192, 0)])
def test_rope_matches_the_rotation(dtype, interleaved, T, H, D, r, off):
    g = torch.Generator(device="cuda").manual_seed(T * 31 + D)
    x = torch.randn(T, H, D, generator=g, device="cuda").to(dtype)
    cs = rt.rope_cos_sin(4096, r, factor=8.0, original_positions=512, device="cuda")
    pos = torch.randint(0, 4096, (T,), generator=g, device="cuda", dtype=torch.int64 if T % 2 else torch.int32)
    for inverse in (False, True):
        want, size = rotated(x, pos, cs, off, interleaved, inverse)
        check(rt.apply_rope(x, pos, cs, off, interleaved, inverse), want, size, dtype)
        y = x.clone()
        assert rt.apply_rope(y, pos, cs, off, interleaved, inverse, out=y) is y
        check(y, want, size, dtype)
    assert rt.device_errors() == 0


def test_rope_strided_views_and_two_dims():
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(9, 4, 200, generator=g, device="cuda").to(torch.bfloat16)
    cs = rt.rope_cos_sin(64, 64, device="cuda")
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    for x in (base[..., 8:136], base[..., 3:131], base.transpose(0, 1)[:, :, :128].transpose(0, 1)[::2], base[:, 1, :96]):
        out = torch.zeros(x.shape[0], *([x.shape[1] + 1] if x.dim() == 3 else []), x.shape[-1] + 8, device="cuda",
                          dtype=torch.bfloat16)
        o = out[:, 1:, 8:] if x.dim() == 3 else out[:, 8:]
        n = x.shape[0]
        rt.apply_rope(x, pos[:n], cs, 0, False, out=o)
        want, size = rotated(x if x.dim() == 3 else x[:, None], pos[:n], cs, 0, False, False)
        check(o if x.dim() == 3 else o[:, None], want, size, torch.bfloat16)
        assert not out[..., :8].any()


def test_rope_gradient_is_the_inverse_and_matches_differences():
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w = (torch.randn(6, 2, 48, generator=g, device="cuda") for _ in range(2))
    cs = rt.rope_cos_sin(100, 32, device="cuda")
    pos = torch.randint(0, 100, (6,), generator=g, device="cuda")
    grad = rt.apply_rope(w, pos, cs, 8, True, inverse=True)
    want, size = rotated(w, pos, cs, 8, True, True)
    check(grad, want, size, torch.float32)
    f = lambda v: float((rt.apply_rope(v, pos, cs, 8, True).double() * w.double()).sum())  # noqa: E731
    for t, h, d in [(0, 0, 0), (1, 1, 8), (2, 0, 9), (3, 1, 39), (5, 0, 40), (4, 1, 47)]:
        e = torch.zeros_like(x)
        e[t, h, d] = 1.0
        # linear in x: the difference quotient is exact up to the fp32 roundings of the outputs it sums
        tol = 8 * 2.0 ** -24 * float((x.abs() + 2).max()) * float(w.abs().sum())
        assert abs((f(x + e) - f(x - e)) / 2 - float(grad[t, h, d])) <= tol


def test_rope_positions_outside_the_table_are_flagged_and_left():
    x = torch.randn(4, 2, 64, device="cuda")
    cs = rt.rope_cos_sin(8, 64, device="cuda")
    pos = torch.tensor([3, 8, -1, 7], device="cuda")
    y = rt.apply_rope(x, pos, cs)
    assert rt.device_errors() == _lib.DEVERR_BAD_INDEX
    assert torch.equal(y[1:3], x[1:3])
    want, size = rotated(x[[0, 3]], pos[[0, 3]], cs, 0, True, False)
    check(y[[0, 3]], want, size, torch.float32)


def test_rope_far_offsets():
    """A tensor whose last row starts past 2^32 elements."""
    H, D = 64, 576
    T = (1 << 32) // (H * D) + 2
    x = torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
    x[-1] = 1.0
    cs = rt.rope_cos_sin(16, 64, device="cuda")
    pos = torch.full((T,), 5, dtype=torch.int32, device="cuda")
    rt.apply_rope(x, pos, cs, out=x)
    want, size = rotated(torch.ones(1, H, D, dtype=torch.bfloat16, device="cuda"), pos[:1], cs, 512, True, False)
    check(x[-1:], want, size, torch.bfloat16)
    assert not x[-2].any()


def test_rope_cos_sin_yarn_blend():
    cs = rt.rope_cos_sin(1 << 17, 64, factor=16.0, original_positions=4096)
    plain = rt.rope_cos_sin(1 << 17, 64)
    gain = 0.1 * math.log(16.0) + 1.0
    # the fastest dim keeps its frequency, the slowest is divided by the factor
    assert torch.allclose(cs[:, 0], gain * plain[:, 0], atol=1e-6)
    assert torch.allclose(cs[:, 31], gain * torch.cos(torch.arange(1 << 17, dtype=torch.float64) * 10000.0 ** (-31 / 32) / 16.0).float(), atol=1e-6)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,H", [(1, 1), (5, 64), (130, 3), (7, 0)])
def test_rotated_rope_rows(interleaved, T, H):
    g = torch.Generator(device="cuda").manual_seed(T + H)
    pages, page = 9, 16
    cache = torch.randn(pages, page, 64, generator=g, device="cuda").to(torch.bfloat16)
    before = cache.clone()
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
    if T > 4:
        slots[2], slots[4] = -1, pages * page
    if T == 130:
        slots = slots.int()
    k = torch.randn(T, 576, generator=g, device="cuda").to(torch.bfloat16)[:, 512:]
    cs = rt.rope_cos_sin(300, 64, device="cuda")
    pos = torch.randint(0, 300, (T,), generator=g, device="cuda", dtype=torch.int32)
    q = torch.randn(T, H, 192, generator=g, device="cuda").to(torch.bfloat16)[..., 128:] if H else None
    out = torch.zeros(T, H, 576, dtype=torch.bfloat16, device="cuda") if H else None
    rt.write_nvfp4_rope_rotated(k, cache, slots, pos, cs, q_pe=q, q_out=out[..., 512:] if H else None,
                                interleaved=interleaved)
    assert rt.device_errors() == (_lib.DEVERR_BAD_SLOT if T > 4 else 0)
    live = (slots >= 0) & (slots < pages * page)
    want, size = rotated(k[:, None], pos, cs, 0, interleaved, False)
    rows = cache.view(-1, 64)
    check(rows[slots[live].long()][:, None], want[live], size[live], torch.bfloat16)
    other = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    other[slots[live].long()] = False
    assert torch.equal(rows[other], before.view(-1, 64)[other])
    if H:
        want, size = rotated(q, pos, cs, 0, interleaved, False)
        check(out[..., 512:], want, size, torch.bfloat16)
        assert not out[..., :512].any()
        q1 = q.clone()
        rt.write_nvfp4_rope_rotated(k, cache, slots.clamp_max(-1), pos, cs, q_pe=q1, interleaved=interleaved)
        assert torch.equal(q1, out[..., 512:])


def test_rotated_rope_rows_unaligned_views():
    g = torch.Generator(device="cuda").manual_seed(9)
    cache = torch.zeros(4, 16, 64, dtype=torch.bfloat16, device="cuda")
    k = torch.randn(6, 67, generator=g, device="cuda").to(torch.bfloat16)[:, 3:]
    q = torch.randn(6, 2, 71, generator=g, device="cuda").to(torch.bfloat16)[..., 7:]
    cs = rt.rope_cos_sin(300, 64, device="cuda")
    pos = torch.randint(0, 300, (6,), generator=g, device="cuda")
    slots = torch.arange(6, device="cuda", dtype=torch.int32) * 7
    rt.write_nvfp4_rope_rotated(k, cache, slots, pos, cs, q_pe=q, q_out=(out := torch.empty(6, 2, 64, dtype=torch.bfloat16, device="cuda")))
    want, size = rotated(k[:, None], pos, cs, 0, True, False)
    check(cache.view(-1, 64)[slots.long()][:, None], want, size, torch.bfloat16)
    want, size = rotated(q, pos, cs, 0, True, False)
    check(out, want, size, torch.bfloat16)
