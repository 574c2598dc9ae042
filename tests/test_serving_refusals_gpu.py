"""GPU: what the serving operators' Python entries refuse, before any launch."""
import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt

pytestmark = pytest.mark.gpu


def bf16(*n):
    return torch.zeros(*n, dtype=torch.bfloat16, device="cuda")


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def pool(pages=4, page=16):
    return torch.zeros(pages, page, 288, dtype=torch.uint8, device="cuda")


def refuses(call, args, change, error, word):
    with pytest.raises(error, match=word):
        call(**(args | change))


@pytest.mark.parametrize("change,error,word", [
    (dict(x=torch.zeros(4, 2, 64)), ValueError, "x must be a CUDA"),
    (dict(x="x"), ValueError, "x must be a CUDA"),
    (dict(x=lambda: torch.zeros(4, 2, 64, dtype=torch.float64, device="cuda")), TypeError, "bfloat16"),
    (dict(x=lambda: bf16(4, 64, 2).transpose(1, 2)), ValueError, "contiguous last"),
    (dict(x=lambda: bf16(64)), ValueError, "T, H, D"),
    (dict(out=lambda: bf16(4, 2, 32)), ValueError, "out must have"),
    (dict(out=lambda: torch.zeros(4, 2, 64, device="cuda")), ValueError, "out must have"),
    (dict(positions=lambda: i32(0, 1, 2)), ValueError, "3 entries for 4"),
    (dict(positions=lambda: torch.zeros(4, device="cuda")), TypeError, "positions"),
    (dict(positions=torch.zeros(4, dtype=torch.int32)), ValueError, "positions must be a CUDA"),
    (dict(cos_sin=lambda: bf16(8, 64)), ValueError, "float32"),
    (dict(cos_sin=lambda: torch.zeros(8, 66, device="cuda")), RuntimeError, "rotary_dim"),
    (dict(rope_offset=1), RuntimeError, "rotary_dim"),
])
def test_apply_rope(change, error, word):
    args = dict(x=bf16(4, 2, 64), positions=i32(0, 1, 2, 3), cos_sin=torch.zeros(8, 64, device="cuda"))
    refuses(rt.apply_rope, args, {k: v() if callable(v) else v for k, v in change.items()}, error, word)


@pytest.mark.parametrize("change,error,word", [
    (dict(k_pe=torch.zeros(4, 64)), ValueError, "k_pe must be a CUDA"),
    (dict(k_pe=lambda: bf16(4, 63)), ValueError, "k_pe must be bf16"),
    (dict(k_pe=lambda: bf16(4, 1, 64)), ValueError, "k_pe must be bf16"),
    (dict(k_pe=lambda: torch.zeros(4, 64, device="cuda")), ValueError, "k_pe must be bf16"),
    (dict(k_pe=lambda: bf16(64, 4).T), ValueError, "k_pe must be bf16"),
    (dict(rope_cache=lambda: torch.zeros(2, 16, 64, device="cuda")), TypeError, "rope_cache"),
    (dict(rope_cache=lambda: bf16(3, 5)), ValueError, "rows of 64"),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int64)), ValueError, "slot_mapping must be a CUDA"),
    (dict(slot_mapping=lambda: i32(0)), ValueError, "1 entries for 4"),
    (dict(slot_mapping=lambda: torch.zeros(4, device="cuda")), TypeError, "slot_mapping"),
    (dict(positions=lambda: i32(0)), ValueError, "1 entries for 4"),
    (dict(cos_sin=lambda: torch.zeros(8, 32, device="cuda")), ValueError, "cos_sin"),
    (dict(q_pe=lambda: bf16(3, 2, 64)), ValueError, "q_pe must be bf16"),
    (dict(q_pe=lambda: bf16(4, 2, 32)), ValueError, "q_pe must be bf16"),
    (dict(q_pe=torch.zeros(4, 2, 64)), ValueError, "q_pe must be a CUDA"),
    (dict(q_pe=lambda: bf16(4, 2, 64), q_out=lambda: bf16(4, 1, 64)), ValueError, "q_out must be"),
    (dict(q_out=lambda: bf16(4, 2, 64)), ValueError, "without q_pe"),
])
def test_rotated_rows(change, error, word):
    args = dict(k_pe=bf16(4, 64), rope_cache=bf16(2, 16, 64), slot_mapping=i32(0, 1, 2, 3), positions=i32(0, 1, 2, 3),
                cos_sin=torch.zeros(8, 64, device="cuda"))
    refuses(rt.write_nvfp4_rope_rotated, args, {k: v() if callable(v) else v for k, v in change.items()}, error, word)


@pytest.mark.parametrize("change,error,word", [
    (dict(query=torch.zeros(2, 2, 576)), ValueError, "query must be a CUDA"),
    (dict(query=None), ValueError, "query must be a CUDA"),
    (dict(block_tables=None), ValueError, "block_tables must be a CUDA"),
    (dict(seq_lens=torch.zeros(1, dtype=torch.int32)), ValueError, "seq_lens must be a CUDA"),
    (dict(rope_cache=torch.zeros(4, 16, 64)), ValueError, "rope_cache must be a CUDA"),
    (dict(bmm1_scale=lambda: torch.ones((), device="cuda")), TypeError, "Python floats"),
    (dict(query=lambda: torch.zeros(2, 2, 576, device="cuda")), ValueError, "query must be bf16"),
    (dict(query=lambda: bf16(2, 1152)), ValueError, "query must be bf16"),
    (dict(query=lambda: bf16(2, 2, 512)), ValueError, "query dim"),
    (dict(kv_lora_rank=256), ValueError, "query dim"),
    (dict(kv_cache=lambda: torch.zeros(4, 16, 656, dtype=torch.uint8, device="cuda")), ValueError, "288-byte"),
    (dict(kv_cache=lambda: pool(8)[::2]), ValueError, "288-byte"),
    (dict(seq_lens=lambda: torch.zeros(1, dtype=torch.int64, device="cuda")), TypeError, "int32"),
    (dict(block_tables=lambda: i32(0, 1)), ValueError, "block_tables must be"),
    (dict(block_tables=lambda: i32(0, 1, 2, 3).view(2, 2)), ValueError, "block_tables must be"),
    (dict(block_tables=lambda: i32(0, 1, 2, 3).view(1, 4)[:, ::2]), ValueError, "block_tables must be"),
    (dict(cu_seqlens_q=lambda: i32(0, 1, 2)), ValueError, "one entry more"),
    (dict(max_seq_len=33), ValueError, "too narrow"),
    (dict(out=lambda: bf16(2, 2, 576)), ValueError, "out must be"),
    (dict(out=torch.zeros(2, 2, 512, dtype=torch.bfloat16)), ValueError, "out must be"),
    (dict(rope_cache=lambda: bf16(3, 16, 64)), ValueError, "side-pool"),
    (dict(query=lambda: bf16(2, 2, 584)[..., 4:580]), RuntimeError, "16-byte aligned"),
    (dict(max_q_len=-1), RuntimeError, "max_q_len"),
])
def test_mla_prefill(change, error, word):
    args = dict(query=bf16(2, 2, 576), kv_cache=pool(), workspace_buffer=None, kv_lora_rank=512, qk_rope_head_dim=64,
                block_tables=i32(0, 1).view(1, 2), cu_seqlens_q=i32(0, 2), seq_lens=i32(20), max_q_len=2, max_seq_len=32)
    refuses(rt.mla_prefill, args, {k: v() if callable(v) else v for k, v in change.items()}, error, word)


def test_page_upkeep():
    caches, tables, seq, refs = [pool(), pool()], i32(0, 1, -1, -1).view(2, 2), i32(20, 0), i32(1, 1, 0, 0)
    src, dst = i32(0), i32(1)
    fork = dict(caches=caches, block_tables=tables, seq_lens=seq, src=src, dst=dst, ref_counts=refs)
    for change, error, word in [
        (dict(caches=[]), ValueError, "at least one"),
        (dict(caches=[pool(), pool(5)]), ValueError, "one geometry"),
        (dict(caches=[pool()] * 9), ValueError, "at most 8"),
        (dict(caches=[pool(8)[::2]]), ValueError, "contiguous"),
        (dict(block_tables=tables.long()), TypeError, "block_tables"),
        (dict(block_tables=tables[0]), ValueError, "block_tables"),
        (dict(seq_lens=i32(20)), ValueError, "one entry per row"),
        (dict(dst=i32(1, 1)), ValueError, "same length"),
        (dict(ref_counts=i32(1, 1)), ValueError, "one per page"),
        (dict(src=torch.zeros(1, dtype=torch.int32)), ValueError, "src must be a CUDA"),
    ]:
        refuses(rt.fork_pages, fork, change, error, word)
    refuses(rt.free_pages, dict(block_tables=tables, seq_lens=seq, slots=src, ref_counts=refs), dict(seq_lens=i32(1)), ValueError, "one entry")
    refuses(rt.copy_pages, dict(caches=caches, src=src, dst=dst), dict(dst=i32(1, 2)), ValueError, "same length")
    for change in (dict(ref_counts=i32(1)), dict(out_tables=i32(1, 2).view(1, 2)), dict(out_ref_counts=i32(0))):
        refuses(rt.compact_pages, dict(caches=caches, block_tables=tables, ref_counts=refs), change, ValueError, "ref_counts must")
    assert rt.device_errors() == 0
    assert tables.tolist() == [[0, 1], [-1, -1]] and seq.tolist() == [20, 0] and refs.tolist() == [1, 1, 0, 0]
