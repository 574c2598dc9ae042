"""GPU: lengths past the bounds that a call gives for them."""
import copy

import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt
from test_mla_prefill_gpu import Problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,ctx,most,H", [([20, 13], [150, 77], 9, 12), ([300, 2], [2000, 700], 33, 64), ([40], [30], 35, 5)])
def test_new_tokens_past_max_q_len_are_left_out_and_flagged(new, ctx, most, H):
    """The first max_q_len new tokens of a sequence see what they see in the whole chunk; the rows of the
    others keep what was in them."""
    p = Problem(new, ctx, H, 16, True, seed=sum(new))
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    seq = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    out = torch.full((sum(new), H, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    out, lse = rt.mla_prefill(p.q, p.pool, None, 512, 64, p.tables.cuda(), cu, seq, most, max(ctx), out=out, bmm1_scale=p.scale,
                              rope_cache=p.rope, return_lse=True)
    assert rt.device_errors() == _lib.DEVERR_SEQ_LEN
    keep = torch.cat([torch.arange(n) < most for n in new]).cuda()
    # the same rows as a chunk that ends with them
    kept = copy.copy(p)
    kept.new = [min(n, most) for n in new]
    kept.ctx = [max(0, c - (n - m)) for n, m, c in zip(new, kept.new, ctx)]
    kept.q = p.q[keep]
    kept.check(out[keep], lse[keep])
    assert bool((out[~keep] == 7.0).all())


def test_a_sequence_past_max_seq_len_ends_there_and_is_flagged():
    p = Problem([20, 13], [150, 77], 12, 16, True, seed=12)
    cu = torch.tensor([0, 20, 33], dtype=torch.int32, device="cuda")
    out, lse = rt.mla_prefill(p.q, p.pool, None, 512, 64, p.tables.cuda(), cu, torch.tensor([150, 400], dtype=torch.int32, device="cuda"),
                              20, 150, bmm1_scale=p.scale, rope_cache=p.rope, return_lse=True)
    assert rt.device_errors() == _lib.DEVERR_SEQ_LEN | _lib.DEVERR_BAD_PAGE      # (tokens 77 .. 149 have no page)
    whole = p.run()
    assert torch.equal(out[:20], whole[0][:20]) and torch.equal(lse[:20], whole[1][:20])


def test_rows_past_the_last_sequence_are_not_written():
    """The padding rows of a captured batch."""
    p = Problem([5, 2], [300, 40], 8, 16, True, seed=2)
    p.q = torch.cat([p.q, torch.full((4, 8, 576), float("nan"), dtype=torch.bfloat16, device="cuda")])
    out = torch.full((11, 8, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    out, lse = p.run(out=out)
    assert rt.device_errors() == 0
    p.check(out[:7], lse[:7])
    assert bool((out[7:] == 7.0).all())
