"""Drop-in NVFP4 KV-pool runtime for B200 (sm_100a).

Same module surface as the reference's ``nvfp4-kv/glm53_nvfp4_runtime.py``
(Plaaasma/glm53-flash-dual-dgx-spark), which the vLLM seam patcher copies into the vLLM
package as ``vllm.glm53_nvfp4_runtime``:

    NV_BYTES, DS_BYTES, enabled(), write_nvfp4(), _gather(), build_scratch(),
    _SYNC_FREE_T, _bufs

plus the fused read path the reference does not have:

    mla_decode(query, kv_cache, workspace_buffer, qk_nope_head_dim, kv_lora_rank,
               qk_rope_head_dim, block_tables, seq_lens, max_seq_len,
               sparse_mla_top_k=0, out=None, bmm1_scale=1.0, bmm2_scale=1.0)

argument-compatible with FlashInfer's ``trtllm_batch_decode_with_kv_cache_mla`` (the
consumer the reference feeds, patch_nvfp4_kv.py:84-118) but reading the 288-byte pool
rows directly instead of a 656-byte fp8 scratch.

Every compute call goes through the C ABI of ``libnvfp4kv.so`` on the current torch CUDA
stream; nothing synchronises the host and nothing falls back to the CPU.
"""
from __future__ import annotations

import ctypes
import math
import os
import struct
from typing import NamedTuple

import torch

from . import _lib

NV_BYTES = 288
DS_BYTES = 656
LATENT = 512
ROPE = 64

_ON = os.environ.get("GLM53_NVFP4_KV", "0") == "1"          # read once at import (runtime:29)

# Sync-free ceiling of build_scratch (runtime:134-140): steps with at most this many query
# tokens gather every table entry into a persistent buffer (no host sync, graph-safe).
_SYNC_FREE_T = int(os.environ.get("GLM53_NVFP4_SYNCFREE_T", "192"))
# The T > _SYNC_FREE_T branch of build_scratch deduplicates on the device
# (build_scratch_sync_free), so no step synchronises the host.  GLM53_NVFP4_UNIQUE=1 restores
# the reference's torch.unique branch (runtime:177-182), which synchronises to size its output.
_UNIQUE = os.environ.get("GLM53_NVFP4_UNIQUE", "0") == "1"
# Rows of the device branch's persistent scratch (656 B each).  0 (default): min(T * K, pool
# rows + 1), the most distinct entries a step can have; a smaller bound caps the memory, and a
# step with more distinct entries than it sets NVFP4KV_DEVERR_CAPACITY.
_SYNC_FREE_ROWS = int(os.environ.get("GLM53_NVFP4_SYNCFREE_ROWS", "0"))

# Division of the 656 B row encoders (_gather, build_scratch): "ieee" (default) gives the
# reference's rows as it computes on the CPU, "triton" its rows as Triton compiles it for the
# GPU (approximate fp32 division), byte for byte.  See set_gather_division.
_GATHER_DIV = os.environ.get("GLM53_NVFP4_GATHER_DIV", "ieee")

# Persistent device buffers keyed like the reference's: ("shared", K, device index) for the
# build_scratch buffer; ("err", index) / ("ws", index) for this module's own state.
_bufs: dict = {}
_ws_sizes: dict = {}   # decode workspace bytes per (batch, q_len, heads, max_seq_len, topk, device)


def enabled() -> bool:
    return _ON


# ------------------------------------------------------------------ helpers
def _stream(dev: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this runtime has no CPU path)")


def _err_word(dev: torch.device) -> torch.Tensor:
    key = ("err", dev.index)
    e = _bufs.get(key)
    if e is None:
        e = torch.zeros(1, dtype=torch.int32, device=dev)
        _bufs[key] = e
    return e


def device_errors(device=None, clear: bool = True) -> int:
    """Read (and by default clear) the device error word: OR of NVFP4KV_DEVERR_* bits.

    Synchronises with the device; meant for tests and health checks, not the hot path.
    """
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    e = _err_word(dev)
    v = int(e.item())
    if clear:
        e.zero_()
    return v


class _on_device:
    """Make `dev` current for the C call when it is not already (launches use it)."""

    def __init__(self, dev: torch.device):
        self.dev = dev
        self.prev = None

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.dev.index:
            self.prev = cur
            torch.cuda.set_device(self.dev)
        return self

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)


# ------------------------------------------------------------------ write path
def write_nvfp4(kv_c: torch.Tensor, kv_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """kv_c [T, 512] -> NVFP4 rows at slot_mapping in kv_cache (viewed [-1, 288]).

    Same contract as the reference (runtime:68-76): T == 0 is a no-op, slots < 0 are
    skipped.  Slots past the pool are skipped too and flagged in the device error word.
    """
    pool = kv_cache.view(-1, NV_BYTES)
    T = kv_c.shape[0]
    if T == 0:
        return
    _require_cuda(kv_c, "kv_c")
    _require_cuda(pool, "kv_cache")
    if kv_c.dtype == torch.bfloat16:
        dt = _lib.DTYPE_BF16
    elif kv_c.dtype == torch.float16:
        dt = _lib.DTYPE_F16
    else:
        raise TypeError(f"kv_c must be bfloat16 or float16, got {kv_c.dtype}")
    if kv_c.dim() != 2 or kv_c.shape[1] < LATENT or kv_c.stride(1) != 1:
        raise ValueError("kv_c must be [T, >=512] with a contiguous last dimension")
    if pool.dtype != torch.uint8:
        raise TypeError("kv_cache must be a uint8 pool")
    slot = slot_mapping.reshape(-1)
    if slot.numel() != T:
        raise ValueError(f"slot_mapping has {slot.numel()} entries for {T} tokens")
    if slot.dtype == torch.int64:
        sdt = _lib.INDEX_I64
    elif slot.dtype == torch.int32:
        sdt = _lib.INDEX_I32
    else:
        raise TypeError("slot_mapping must be int64 or int32")
    slot = slot.contiguous()
    dev = kv_c.device
    with _on_device(dev):
        rc = _lib.lib().nvfp4kv_append(kv_c.data_ptr(), dt, T, kv_c.stride(0), pool.data_ptr(),
                                       pool.shape[0], slot.data_ptr(), sdt,
                                       _err_word(dev).data_ptr(), _stream(dev))
    _lib.check(rc, "nvfp4kv_append")


def write_nvfp4_rope(k_pe: torch.Tensor, rope_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """k_pe [T, 64] bf16 -> the rope side-pool rope_cache (any shape, 64 bf16 per token slot) at
    slot_mapping; slots < 0 are skipped.  Not in the reference, which drops k_pe for its NoPE
    model (patch_nvfp4_kv.py:70); for MLA models that keep a rope part, beside write_nvfp4."""
    T = k_pe.shape[0]
    if T == 0:
        return
    _require_cuda(k_pe, "k_pe")
    _require_cuda(rope_cache, "rope_cache")
    if k_pe.dtype != torch.bfloat16 or k_pe.dim() != 2 or k_pe.shape[1] < ROPE or k_pe.stride(1) != 1:
        raise ValueError("k_pe must be bf16 [T, >=64] with a contiguous last dimension")
    rope = rope_cache.view(-1, ROPE)
    if rope.dtype != torch.bfloat16:
        raise TypeError("rope_cache must be bf16")
    slot = slot_mapping.reshape(-1).contiguous()
    if slot.numel() != T:
        raise ValueError(f"slot_mapping has {slot.numel()} entries for {T} tokens")
    sdt = _lib.INDEX_I64 if slot.dtype == torch.int64 else _lib.INDEX_I32 if slot.dtype == torch.int32 else None
    if sdt is None:
        raise TypeError("slot_mapping must be int64 or int32")
    dev = k_pe.device
    with _on_device(dev):
        rc = _lib.lib().nvfp4kv_append_rope(k_pe.data_ptr(), T, k_pe.stride(0), rope.data_ptr(), rope.shape[0],
                                            slot.data_ptr(), sdt, _err_word(dev).data_ptr(), _stream(dev))
    _lib.check(rc, "nvfp4kv_append_rope")


# ------------------------------------------------------------------ 656-byte read path
def set_gather_division(mode: str) -> None:
    """Division of the 656-byte row encoders, process-wide: "ieee" (exact; the reference's
    _gather_kernel as it computes on the CPU) or "triton" (div.full.f32, the approximate fp32
    division GPU Triton compiles the reference's `amax / 448.0` and `1.0 / gscale` to, so the
    rows are byte-identical to the reference's GPU output).  No counterpart in the reference."""
    modes = {"ieee": _lib.DIV_IEEE, "triton": _lib.DIV_TRITON}
    if mode not in modes:
        raise ValueError(f"gather division must be 'ieee' or 'triton', got {mode!r}")
    _lib.check(_lib.lib().nvfp4kv_set_gather_division(modes[mode]), "nvfp4kv_set_gather_division")


def get_gather_division() -> str:
    return "triton" if _lib.lib().nvfp4kv_get_gather_division() == _lib.DIV_TRITON else "ieee"


if _GATHER_DIV != "ieee":
    set_gather_division(_GATHER_DIV)


def _gather(pool: torch.Tensor, idx: torch.Tensor, out: torch.Tensor, rope: torch.Tensor | None = None) -> None:
    """NVFP4 pool rows at idx -> fp8_ds_mla 656-byte rows in out (runtime:128-131).  With a rope
    side-pool ``rope`` (not in the reference) the rows' rope bytes carry its 64 bf16."""
    S = idx.shape[0]
    if S == 0:
        return
    _require_cuda(pool, "pool")
    if idx.dtype != torch.int32:
        raise TypeError("idx must be int32")
    if out.dtype != torch.uint8 or out.shape[-1] != DS_BYTES or not out.is_contiguous():
        raise ValueError("out must be a contiguous [S, 656] uint8 tensor")
    idx = idx.contiguous()
    dev = pool.device
    with _on_device(dev):
        if rope is None:
            rc = _lib.lib().nvfp4kv_gather_ds656(pool.data_ptr(), pool.shape[0], idx.data_ptr(), S,
                                                 out.data_ptr(), _stream(dev))
        else:
            r = rope.reshape(-1, ROPE)
            if r.dtype != torch.bfloat16 or r.shape[0] != pool.shape[0] or not r.is_contiguous():
                raise ValueError("rope must be a contiguous bf16 [pool rows, 64] side-pool")
            rc = _lib.lib().nvfp4kv_gather_ds656_rope(pool.data_ptr(), r.data_ptr(), pool.shape[0], idx.data_ptr(),
                                                      S, out.data_ptr(), _stream(dev))
    _lib.check(rc, "nvfp4kv_gather_ds656")


def build_scratch(kv_cache: torch.Tensor, block_tables: torch.Tensor):
    """kv_cache: allocated pool (any shape, 288 B/token rows).
    block_tables: [T, 1, K] int32 physical token rows (-1 padded).
    Returns (scratch [P, 64, 656] uint8, tables [T, 1, K] into scratch), as the reference
    (runtime:143-182): T <= _SYNC_FREE_T gathers every entry into a persistent buffer with
    fixed shapes and no host sync.  Larger T deduplicates on the device without a host sync
    (build_scratch_sync_free): the tables equal the reference's, and the reference's
    ceil(n_unique / 64) pages are the first pages of a persistent capacity-sized scratch (the
    consumer reads only the rows the tables name).  With GLM53_NVFP4_UNIQUE=1 the large branch
    is the reference's torch.unique one, which synchronises the host.
    """
    pool = kv_cache.view(-1, NV_BYTES)
    T, one, K = block_tables.shape
    flat = block_tables.view(-1)
    dev = pool.device
    if T <= _SYNC_FREE_T:
        S = T * K
        P = (S + 63) // 64
        key = ("shared", K, dev.index)
        ent = _bufs.get(key)
        if ent is None:
            pcap = (_SYNC_FREE_T * K + 63) // 64
            ent = (torch.zeros(pcap, 64, DS_BYTES, dtype=torch.uint8, device=dev),
                   torch.arange(pcap * 64, dtype=torch.int32, device=dev))
            _bufs[key] = ent
        buf, ar = ent
        _gather(pool, flat, buf.view(-1, DS_BYTES)[:S])
        return buf[:P], ar[:S].view(T, 1, K)
    if not _UNIQUE:
        scratch, tables, _ = build_scratch_sync_free(kv_cache, block_tables,
                                                     capacity_rows=_SYNC_FREE_ROWS or None)
        return scratch, tables
    uniq, inv = torch.unique(flat, return_inverse=True)
    S = uniq.shape[0]
    P = (S + 63) // 64
    scratch = torch.zeros(P, 64, DS_BYTES, dtype=torch.uint8, device=dev)
    _gather(pool, uniq.to(torch.int32), scratch.view(-1, DS_BYTES)[:S])
    return scratch, inv.to(torch.int32).view(T, 1, K)


def build_scratch_sync_free(kv_cache: torch.Tensor, block_tables: torch.Tensor,
                            capacity_rows: int | None = None):
    """The T > _SYNC_FREE_T branch of build_scratch without a host synchronisation.

    The reference deduplicates with torch.unique (runtime:177-182), which synchronises to
    size its output.  Here the distinct entries are found, numbered in ascending order and
    gathered on the device by fixed-size launches (nvfp4kv_dedup_gather_ds656), so the call
    is asynchronous and CUDA-graph capturable.  Returns (scratch [P_cap, 64, 656] uint8,
    tables [T, 1, K] int32, n_unique int32 [1] on the device).  tables equals the
    reference's; the reference's scratch is the first ceil(n_unique / 64) pages of this one
    (rows from n_unique to the end of that page are zero); later pages are not written.
    P_cap covers capacity_rows rows, by default min(T * K, pool rows + 1), the most distinct
    entries there can be; fewer rows than the distinct entries set NVFP4KV_DEVERR_CAPACITY.
    The scratch is a view of one persistent buffer per device, allocated when a call needs
    more rows than it holds (656 B per row; for a 2,713,846-row pool and 2048 x 2048 entries
    the default capacity is 2,713,847 rows = 1.78 GB) and overwritten by the next call, like
    the reference's persistent sync-free buffer.
    """
    pool = kv_cache.view(-1, NV_BYTES)
    _require_cuda(pool, "kv_cache")
    _require_cuda(block_tables, "block_tables")
    if block_tables.dim() != 3:
        raise ValueError("block_tables must be [T, 1, K]")
    if block_tables.dtype != torch.int32:
        raise TypeError("block_tables must be int32")
    T, one, K = block_tables.shape
    flat = block_tables.reshape(-1).contiguous()
    n = flat.numel()
    R = pool.shape[0]
    cap = min(n, R + 1) if capacity_rows is None else int(capacity_rows)
    if cap < 0:
        raise ValueError("capacity_rows must be >= 0")
    dev = pool.device
    P = (cap + 63) // 64
    skey = ("dedup_scratch", dev.index)
    buf = _bufs.get(skey)
    if buf is None or buf.shape[0] < P:
        _bufs.pop(skey, None)
        buf = torch.empty(P, 64, DS_BYTES, dtype=torch.uint8, device=dev)
        _bufs[skey] = buf
    scratch = buf[:P]
    tables = torch.empty(n, dtype=torch.int32, device=dev)
    n_unique = torch.empty(1, dtype=torch.int32, device=dev)
    ints = ctypes.c_int64()
    _lib.check(_lib.lib().nvfp4kv_dedup_workspace_ints(R, n, ctypes.byref(ints)), "nvfp4kv_dedup_workspace_ints")
    key = ("dedup", dev.index)
    ws = _bufs.get(key)
    if ws is None or ws.numel() < ints.value:
        ws = torch.empty(ints.value, dtype=torch.int32, device=dev)
        _bufs[key] = ws
    with _on_device(dev):
        rc = _lib.lib().nvfp4kv_dedup_gather_ds656(pool.data_ptr(), R, flat.data_ptr(), n, ws.data_ptr(),
                                                   ws.numel(), tables.data_ptr(), scratch.data_ptr(), P * 64,
                                                   n_unique.data_ptr(), _err_word(dev).data_ptr(), _stream(dev))
    _lib.check(rc, "nvfp4kv_dedup_gather_ds656")
    return scratch, tables.view(T, 1, K), n_unique


def dequant(kv_cache: torch.Tensor, rows: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Pool rows -> bf16 [n, 512] (exact); rows outside the pool (and -1) read as zeros."""
    pool = kv_cache.view(-1, NV_BYTES)
    rows = rows.reshape(-1)
    n = rows.numel()
    if out is None:
        out = torch.empty(n, LATENT, dtype=torch.bfloat16, device=pool.device)
    if n == 0:
        return out
    _require_cuda(pool, "kv_cache")
    if rows.dtype == torch.int64:
        rdt = _lib.INDEX_I64
    elif rows.dtype == torch.int32:
        rdt = _lib.INDEX_I32
    else:
        raise TypeError("rows must be int64 or int32")
    if out.dtype != torch.bfloat16 or not out.is_contiguous() or out.numel() < n * LATENT:
        raise ValueError("out must be a contiguous bf16 [n, 512] tensor")
    rows = rows.contiguous()
    dev = pool.device
    with _on_device(dev):
        rc = _lib.lib().nvfp4kv_dequant_bf16(pool.data_ptr(), pool.shape[0], rows.data_ptr(), rdt, n,
                                             out.data_ptr(), _err_word(dev).data_ptr(), _stream(dev))
    _lib.check(rc, "nvfp4kv_dequant_bf16")
    return out


# ------------------------------------------------------------------ fused read path
def mla_decode_workspace_size(batch: int, q_len: int, num_heads: int, max_seq_len: int,
                              sparse_mla_top_k: int = 0, device=None) -> int:
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    out = ctypes.c_size_t(0)
    with _on_device(dev):
        rc = _lib.lib().nvfp4kv_mla_decode_workspace_size(batch, q_len, num_heads, max_seq_len,
                                                          sparse_mla_top_k, ctypes.byref(out))
    _lib.check(rc, "nvfp4kv_mla_decode_workspace_size")
    return int(out.value)


def mla_decode_plan(batch: int, q_len: int, num_heads: int, max_seq_len: int,
                    sparse_mla_top_k: int = 0, device=None) -> tuple[int, int]:
    """(token splits per 64-row query group, kernel launches per mla_decode call)."""
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    splits, launches = ctypes.c_int(0), ctypes.c_int(0)
    with _on_device(dev):
        rc = _lib.lib().nvfp4kv_mla_decode_plan(batch, q_len, num_heads, max_seq_len, sparse_mla_top_k,
                                                ctypes.byref(splits), ctypes.byref(launches))
    _lib.check(rc, "nvfp4kv_mla_decode_plan")
    return int(splits.value), int(launches.value)


def set_kernel_events(start: torch.cuda.Event | None, stop: torch.cuda.Event | None) -> None:
    """Make the calling thread's next mla_decode record `start` / `stop` immediately around its
    attention kernel (a measurement hook; both None clears it)."""
    for e in (start, stop):
        if e is not None and not e.cuda_event:
            e.record()   # torch creates the CUDA event on first record; the library re-records it
    _lib.check(_lib.lib().nvfp4kv_set_kernel_events(
        ctypes.c_void_p(start.cuda_event) if start is not None else None,
        ctypes.c_void_p(stop.cuda_event) if stop is not None else None), "nvfp4kv_set_kernel_events")


def _workspace(dev: torch.device, nbytes: int, given: torch.Tensor | None) -> torch.Tensor | None:
    if nbytes == 0:
        return None
    if given is not None and given.is_cuda and given.numel() * given.element_size() >= nbytes \
            and given.data_ptr() % 256 == 0 and given.is_contiguous():
        return given
    key = ("ws", dev.index)
    ws = _bufs.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=dev)
        _bufs[key] = ws
    return ws


def mla_decode(query: torch.Tensor, kv_cache: torch.Tensor, workspace_buffer: torch.Tensor | None,
               qk_nope_head_dim: int, kv_lora_rank: int, qk_rope_head_dim: int,
               block_tables: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int,
               sparse_mla_top_k: int = 0, out: torch.Tensor | None = None,
               bmm1_scale: float = 1.0, bmm2_scale: float = 1.0,
               rope_cache: torch.Tensor | None = None) -> torch.Tensor:
    """Fused NVFP4 gather + MLA decode (see module docstring).

    query: [B, q_len, H, kv_lora_rank + qk_rope_head_dim] bf16.
    kv_cache: the 288-byte pool, [num_pages, page_size, 288] (or [num_pages, 1, page_size,
      288]); page_size is read from dim -2.
    Dense (sparse_mla_top_k == 0): block_tables [B, max_pages] page ids, seq_lens = context
      lengths.  Sparse: block_tables [B, 1, K] or [B, K] physical token rows (-1 padded),
      seq_lens = number of leading entries to use.
    Returns out [B, q_len, H, kv_lora_rank] bf16.  ``workspace_buffer`` is used for the
    split partials when it is large enough, else a persistent per-device buffer is.
    rope_cache (not in the reference, whose model is NoPE): the rope side-pool, [num_pages,
    page_size, 64] bf16 written by write_nvfp4_rope; the query's last 64 dims then meet it.
    """
    del qk_nope_head_dim  # accepted for signature compatibility; the absorbed MLA form ignores it
    return _decode(query, kv_cache, workspace_buffer, kv_lora_rank, qk_rope_head_dim, block_tables,
                   seq_lens, max_seq_len, sparse_mla_top_k, out, bmm1_scale, bmm2_scale, None, rope_cache)


def mla_decode_lse(query: torch.Tensor, kv_cache: torch.Tensor, workspace_buffer: torch.Tensor | None,
                   qk_nope_head_dim: int, kv_lora_rank: int, qk_rope_head_dim: int,
                   block_tables: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int,
                   sparse_mla_top_k: int = 0, out: torch.Tensor | None = None,
                   bmm1_scale: float = 1.0, bmm2_scale: float = 1.0):
    """mla_decode that also returns lse [B, q_len, H] float32: the natural log of the sum over
    the visible tokens of exp(bmm1_scale * q.k) (-inf for a row that sees no token).  Results of
    disjoint token ranges of one sequence merge exactly through it (see ``partition``).
    Returns (out, lse).  No counterpart in the reference; used by the multi-GPU partition."""
    del qk_nope_head_dim
    B, QL, H = query.shape[0], query.shape[1], query.shape[2]
    lse = torch.empty(B, QL, H, dtype=torch.float32, device=query.device)
    out = _decode(query, kv_cache, workspace_buffer, kv_lora_rank, qk_rope_head_dim, block_tables,
                  seq_lens, max_seq_len, sparse_mla_top_k, out, bmm1_scale, bmm2_scale, lse)
    return out, lse


def _decode(query, kv_cache, workspace_buffer, kv_lora_rank, qk_rope_head_dim, block_tables,
            seq_lens, max_seq_len, sparse_mla_top_k, out, bmm1_scale, bmm2_scale, lse, rope_cache=None):
    _require_cuda(query, "query")
    _require_cuda(kv_cache, "kv_cache")
    if isinstance(bmm1_scale, torch.Tensor) or isinstance(bmm2_scale, torch.Tensor):
        raise TypeError("bmm1_scale / bmm2_scale must be Python floats (a device scalar would need a sync)")
    if query.dtype != torch.bfloat16 or query.dim() != 4:
        raise ValueError("query must be a 4-D bf16 tensor [B, q_len, H, D]")
    if query.stride(3) != 1:
        raise ValueError("query's last dimension must be contiguous")
    B, QL, H, D = query.shape
    if kv_lora_rank != LATENT or D != kv_lora_rank + qk_rope_head_dim:
        raise ValueError(f"query dim {D} must equal kv_lora_rank (512) + qk_rope_head_dim")
    pool = kv_cache.view(-1, NV_BYTES)
    page_size = kv_cache.shape[-2] if kv_cache.dim() >= 3 else 64
    sparse = int(sparse_mla_top_k) > 0
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_tables and seq_lens must be int32")
    bt = block_tables.reshape(B, -1) if sparse else block_tables
    if bt.dim() != 2 or bt.stride(1) != 1:
        raise ValueError("block_tables must be [B, width] with a contiguous last dimension")
    if sparse and bt.shape[1] < sparse_mla_top_k:
        raise ValueError("sparse block_tables narrower than sparse_mla_top_k")
    if not sparse and bt.shape[1] * page_size < max_seq_len:
        raise ValueError("block_tables too narrow for max_seq_len")
    sl = seq_lens.contiguous()
    if out is None:
        out = torch.empty(B, QL, H, LATENT, dtype=torch.bfloat16, device=query.device)
    elif out.shape != (B, QL, H, LATENT) or out.dtype != torch.bfloat16 or out.stride(3) != 1:
        raise ValueError("out must be bf16 [B, q_len, H, 512] with a contiguous last dimension")
    rope = None
    if rope_cache is not None:
        if lse is not None:
            raise ValueError("mla_decode_lse has no rope variant")
        _require_cuda(rope_cache, "rope_cache")
        rope = rope_cache.reshape(-1, ROPE)
        if rope.dtype != torch.bfloat16 or rope.shape[0] != pool.shape[0] or not rope.is_contiguous():
            raise ValueError("rope_cache must be a contiguous bf16 [pool rows, 64] side-pool")
    dev = query.device
    with _on_device(dev):
        size_key = (B, QL, H, int(max_seq_len), int(sparse_mla_top_k), dev.index, rope is not None)
        ws_need = _ws_sizes.get(size_key)
        if ws_need is None:                      # the plan depends only on these and the device
            if rope is None:
                ws_need = mla_decode_workspace_size(B, QL, H, max_seq_len, int(sparse_mla_top_k), dev)
            else:
                n = ctypes.c_size_t(0)
                _lib.check(_lib.lib().nvfp4kv_mla_decode_rope_workspace_size(
                    B, QL, H, int(max_seq_len), int(sparse_mla_top_k), ctypes.byref(n)),
                    "nvfp4kv_mla_decode_rope_workspace_size")
                ws_need = int(n.value)
            _ws_sizes[size_key] = ws_need
        ws = _workspace(dev, ws_need, workspace_buffer)
        args = [query.data_ptr(), query.stride(0), query.stride(1), query.stride(2),
                pool.data_ptr(), pool.shape[0],
                bt.data_ptr(), bt.stride(0), sl.data_ptr(),
                B, QL, H, D, kv_lora_rank,
                int(sparse_mla_top_k), int(page_size), int(max_seq_len),
                float(bmm1_scale), float(bmm2_scale),
                out.data_ptr(), out.stride(0), out.stride(1), out.stride(2)]
        tail = [ws.data_ptr() if ws is not None else None, ws_need, _err_word(dev).data_ptr(), _stream(dev)]
        if rope is not None:
            rc = _lib.lib().nvfp4kv_mla_decode_rope(*args[:6], rope.data_ptr(), *args[6:], *tail)
        elif lse is None:
            rc = _lib.lib().nvfp4kv_mla_decode(*args, *tail)
        else:
            rc = _lib.lib().nvfp4kv_mla_decode_lse(*args, lse.data_ptr(), *tail)
    _lib.check(rc, "nvfp4kv_mla_decode")
    return out


# ------------------------------------------------------------------ indexer K-pool
INDEX_DIM = 128
INDEX_ROW_BYTES = 72


def index_append(k: torch.Tensor, index_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Indexer keys k [T, 128] bf16 -> NVFP4 72-byte rows of index_cache (any shape, 72 bytes per
    token slot) at slot_mapping; slots < 0 are skipped.  The reference keeps its indexer keys in
    an fp8 pool (PLAN.md:29); this is the FP4 pool its README (:321) leaves to sm_100."""
    T = k.shape[0]
    if T == 0:
        return
    _require_cuda(k, "k")
    _require_cuda(index_cache, "index_cache")
    if k.dtype != torch.bfloat16 or k.dim() != 2 or k.shape[1] < INDEX_DIM or k.stride(1) != 1:
        raise ValueError("k must be bf16 [T, >=128] with a contiguous last dimension")
    pool = index_cache.view(-1, INDEX_ROW_BYTES)
    if pool.dtype != torch.uint8:
        raise TypeError("index_cache must be uint8")
    slot = slot_mapping.reshape(-1).contiguous()
    if slot.numel() != T:
        raise ValueError(f"slot_mapping has {slot.numel()} entries for {T} tokens")
    sdt = _lib.INDEX_I64 if slot.dtype == torch.int64 else _lib.INDEX_I32 if slot.dtype == torch.int32 else None
    if sdt is None:
        raise TypeError("slot_mapping must be int64 or int32")
    dev = k.device
    with _on_device(dev):
        rc = _lib.lib().nvfp4kv_index_append(k.data_ptr(), T, k.stride(0), pool.data_ptr(), pool.shape[0],
                                             slot.data_ptr(), sdt, _err_word(dev).data_ptr(), _stream(dev))
    _lib.check(rc, "nvfp4kv_index_append")


def index_topk(q: torch.Tensor, weights: torch.Tensor, index_cache: torch.Tensor, block_tables: torch.Tensor,
               seq_lens: torch.Tensor, max_seq_len: int, topk: int = 2048,
               out_rows: torch.Tensor | None = None, out_count: torch.Tensor | None = None):
    """The DSA indexer's selection over the NVFP4 indexer pool: per entry b, the pool rows of the
    topk positions s < seq_lens[b] with the highest sum_h weights[b, h] * max(q[b, h] . k[s], 0),
    in ascending position order (-1 padded), and their count min(seq_lens[b], topk).
    q [B, 64, 128] bf16, weights [B, 64] fp32, block_tables [B, pages] page ids.  The two
    results are the sparse tables and seq_lens mla_decode(..., sparse_mla_top_k=topk) takes.
    No host synchronisation; the score workspace is a persistent per-device buffer."""
    _require_cuda(q, "q")
    B = q.shape[0]
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[2] != INDEX_DIM or q.stride(2) != 1:
        raise ValueError("q must be bf16 [B, 64, 128] with a contiguous last dimension")
    if weights.dtype != torch.float32 or weights.shape[0] != B or weights.stride(1) != 1:
        raise ValueError("weights must be float32 [B, 64]")
    pool = index_cache.view(-1, INDEX_ROW_BYTES)
    page_size = index_cache.shape[-2] if index_cache.dim() >= 3 else 64
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_tables and seq_lens must be int32")
    dev = q.device
    if out_rows is None:
        out_rows = torch.empty(B, topk, dtype=torch.int32, device=dev)
    if out_count is None:
        out_count = torch.empty(B, dtype=torch.int32, device=dev)
    with _on_device(dev):
        need = ctypes.c_size_t(0)
        _lib.check(_lib.lib().nvfp4kv_index_topk_workspace_size(B, int(max_seq_len), ctypes.byref(need)),
                   "nvfp4kv_index_topk_workspace_size")
        key = ("index_ws", dev.index)
        ws = _bufs.get(key)
        if ws is None or ws.numel() < need.value:
            ws = torch.empty(max(need.value, 1 << 16), dtype=torch.uint8, device=dev)
            _bufs[key] = ws
        rc = _lib.lib().nvfp4kv_index_topk(q.data_ptr(), q.stride(0), q.stride(1), weights.data_ptr(),
                                           weights.stride(0), pool.data_ptr(), pool.shape[0],
                                           block_tables.data_ptr(), block_tables.stride(0),
                                           seq_lens.contiguous().data_ptr(), B, q.shape[1], int(page_size),
                                           int(max_seq_len), int(topk), out_rows.data_ptr(), out_count.data_ptr(),
                                           ws.data_ptr(), ws.numel(), _err_word(dev).data_ptr(), _stream(dev))
    _lib.check(rc, "nvfp4kv_index_topk")
    return out_rows, out_count


def index_scores_buffer(device=None) -> torch.Tensor | None:
    """The score workspace of the last index_topk on `device` (float32, [B, ceil(max_seq_len /
    128) * 128] row-major), for inspection."""
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    ws = _bufs.get(("index_ws", dev.index))
    return None if ws is None else ws.view(torch.float32)


# ------------------------------------------------------------------ serving operators: the call
# A few tokens' operators run for less time on the device than their call takes on the host, so the
# call below uses torch's raw getters, 3 us less than the stream object and device guard, and packs its
# arguments: 2 us less than converting 23 of them one by one (a step of 16 tokens through apply_rope
# 9.4 -> 7.5 us), 3 us for the 30 of mla_prefill.
_raw_stream = torch._C._cuda_getCurrentRawStream


_entries: dict = {}    # C entries by name: the packed call and what it takes


def _call(name: str, index: int, *args) -> None:
    """The C entry ``name`` on device ``index``'s current stream, with the device error word; raises
    on a non-OK code.  Null pointers are 0."""
    word = _bufs.get(("err", index))
    err = (_err_word(torch.device("cuda", index)) if word is None else word).data_ptr()
    entry = _entries.get(name)
    if entry is None:
        entry = _entries[name] = (_lib.lib().nvfp4kv_call_packed, *_lib.packed(name))
    call, number, num, pack = entry
    try:
        words = pack(*args, err, _raw_stream(index))
    except struct.error as e:
        raise TypeError(f"{name}: {e}") from None
    if torch._C._cuda_getDevice() == index:
        rc = call(number, num, words)
    else:
        with _on_device(torch.device("cuda", index)):
            rc = call(number, num, words)
    if rc:
        _lib.check(rc, name)


def _require_on(index: int, t: torch.Tensor, name: str) -> None:
    """t is on CUDA device ``index``: a kernel that reads another device's memory may fault."""
    if not isinstance(t, torch.Tensor) or t.get_device() != index:
        _require_cuda(t, name)
        raise ValueError(f"{name} must be on cuda:{index} like the others")


def _whole(x, name: str) -> int:
    """x as an int that is equal to it (half a token cut off a window would be none at all)."""
    n = int(x)
    if n != x:
        raise TypeError(f"{name} must be whole numbers, not {x!r}")
    return n


def _vector(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() == 1 and t.is_contiguous() else t.reshape(-1).contiguous()


# ------------------------------------------------------------------ rotary positions
_ROPE_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
_INDEX_DTYPES = {torch.int64: _lib.INDEX_I64, torch.int32: _lib.INDEX_I32}


def rope_cos_sin(max_positions: int, rotary_dim: int = ROPE, base: float = 10000.0, factor: float = 1.0,
                 original_positions: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 attention_factor: float | None = None, device=None) -> torch.Tensor:
    """The cos | sin table of the rotary operators, float32 [max_positions, rotary_dim], computed
    in float64.  ``factor`` > 1 stretches the positions for long contexts: by it alone
    (position interpolation), or, with ``original_positions`` (the trained length), by the YaRN
    rule: dims that turn more than ``beta_fast`` times over the trained length keep their
    frequency, those that turn less than ``beta_slow`` times are divided by ``factor``, the ones
    between (their range rounded outwards to whole dims) are blended linearly, and cos and sin
    carry ``attention_factor`` (default 0.1 ln(factor) + 1)."""
    if rotary_dim < 2 or rotary_dim % 2 or max_positions < 1:
        raise ValueError("rotary_dim must be even and >= 2, max_positions >= 1")
    half = rotary_dim // 2
    inv = base ** (-torch.arange(half, dtype=torch.float64) / half)
    gain = 1.0
    if factor != 1.0 and original_positions is None:
        inv = inv / factor
    elif factor != 1.0:
        def dim_of(turns):      # the dim that turns `turns` times over the trained length
            return half * math.log(original_positions / (turns * 2 * math.pi)) / math.log(base)

        # (hi may lie past the last dim: a long trained length leaves the ramp unfinished there)
        lo, hi = max(math.floor(dim_of(beta_fast)), 0), min(math.ceil(dim_of(beta_slow)), rotary_dim - 1)
        blend = ((torch.arange(half, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv * (1 - blend) + inv / factor * blend
        gain = 0.1 * math.log(factor) + 1.0 if attention_factor is None else attention_factor
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * inv.to(device)
    return (torch.cat([angle.cos(), angle.sin()], 1) * gain).float()


def rope_axes(sections, rotary_dim: int = ROPE, dealt: bool = False) -> tuple[int, ...]:
    """The axis of each of the rotary_dim / 2 pairs, for ``axes`` of the rotary operators: sections[a]
    pairs turn by axis a (time, height, width ...; at most 4), in sections one after the other, or
    ``dealt``: a pair to each axis in turn that has some left."""
    left = [_whole(n, "sections") for n in sections]
    if not 1 <= len(left) <= _lib.MAX_AXES or min(left) < 0 or 2 * sum(left) != rotary_dim:
        raise ValueError(f"sections must be 1 to {_lib.MAX_AXES} numbers of pairs that add up to rotary_dim / 2")
    if not dealt:
        return tuple(a for a, n in enumerate(left) for _ in range(n))
    out = []
    while len(out) < rotary_dim // 2:
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] = n - 1
    return tuple(out)


_pair_axes: dict = {}      # the C entries' pair_axes, by the tuple of axes


def _axes(axes, num: int, rotary_dim: int):
    """The host array of a call's pair axes."""
    array = _pair_axes.get((axes, num, rotary_dim)) if type(axes) is tuple else None
    if array is None:
        axes = tuple(_whole(a, "axes") for a in axes)
        if len(axes) != rotary_dim // 2 or not all(0 <= a < num for a in axes):
            raise ValueError(f"axes must be {rotary_dim // 2} numbers in [0, {num}), one for each rotated pair")
        if len(_pair_axes) >= 256:
            _pair_axes.clear()
        array = _pair_axes[axes, num, rotary_dim] = (ctypes.c_uint8 * len(axes))(*axes)
    return array


def _check_axes(index: int, cos_sin: torch.Tensor, positions: torch.Tensor, T: int, rotary_dim: int, axes):
    """_check_angles for positions [axes, T]: also their stride, their number and the pairs' axes."""
    if not (isinstance(positions, torch.Tensor) and positions.get_device() == index == cos_sin.get_device()
            and cos_sin.dtype is torch.float32 and cos_sin.is_contiguous()):
        _check_angles(index, cos_sin, positions, T, rotary_dim)
    shape, st, dtype = positions.shape, positions.stride(), _INDEX_DTYPES.get(positions.dtype)
    if len(shape) != 2 or not 1 <= shape[0] <= _lib.MAX_AXES or shape[1] != T:
        raise ValueError(f"positions must be [axes, {T}] with at most {_lib.MAX_AXES} axes")
    if rotary_dim != cos_sin.shape[1] or rotary_dim > _lib.MAX_AXES_DIM:
        raise ValueError(f"cos_sin must be [positions, {rotary_dim}], with several axes at most {_lib.MAX_AXES_DIM} wide")
    if dtype is None:
        raise TypeError("positions must be int64 or int32")
    if st[1] != 1 and T > 1:
        positions = positions.contiguous()
        st = positions.stride()
    return positions, dtype, st[0], shape[0], _axes(axes, shape[0], rotary_dim)


def _check_angles(index: int, cos_sin: torch.Tensor, positions: torch.Tensor, T: int, rotary_dim: int):
    _require_on(index, cos_sin, "cos_sin")
    _require_on(index, positions, "positions")
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or cos_sin.shape[1] != rotary_dim \
            or not cos_sin.is_contiguous():
        raise ValueError(f"cos_sin must be a contiguous float32 [positions, {rotary_dim}] table")
    pos = _vector(positions)
    if pos.shape[0] != T:
        raise ValueError(f"positions has {pos.shape[0]} entries for {T} tokens")
    dtype = _INDEX_DTYPES.get(pos.dtype)
    if dtype is None:
        raise TypeError("positions must be int64 or int32")
    return pos, dtype


def apply_rope(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, rope_offset: int | None = None,
               interleaved: bool = True, inverse: bool = False, out: torch.Tensor | None = None,
               axes=None) -> torch.Tensor:
    """Rotary positions: x [T, H, D] or [T, D] (bf16, fp16 or fp32, last dim contiguous), dims
    [rope_offset, rope_offset + cos_sin.shape[1]) of every head rotated by its token's angles
    (default: the last dims), the others copied.  ``interleaved`` pairs dims (2i, 2i + 1), else
    (i, i + half).  ``inverse`` rotates back: the gradient with respect to x.  ``out`` may be x;
    a position outside the table leaves its token as it is and is flagged in the device error
    word.  cos_sin: see rope_cos_sin.

    With ``axes`` (the axis of each of the cos_sin.shape[1] / 2 pairs, see rope_axes) positions is
    [axes, T]: pair i of token t turns by positions[axes[i], t]."""
    _require_cuda(x, "x")
    dtype = _ROPE_DTYPES.get(x.dtype)
    if dtype is None:
        raise TypeError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    shape, st = x.shape, x.stride()
    if len(shape) not in (2, 3) or st[-1] != 1:
        raise ValueError("x must be [T, H, D] or [T, D] with a contiguous last dimension")
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
    index = x.get_device()
    _require_on(index, out, "out")
    ost = out.stride()
    if out.shape != shape or out.dtype != x.dtype or ost[-1] != 1:
        raise ValueError("out must have x's shape and dtype and a contiguous last dimension")
    T, D = shape[0], shape[-1]
    H, sh, osh = (shape[1], st[1], ost[1]) if len(shape) == 3 else (1, D, D)
    P, r = cos_sin.shape
    if axes is not None:
        pos, pdt, ps, A, pairs = _check_axes(index, cos_sin, positions, T, r, axes)
        if T and H:
            _call("nvfp4kv_rope_axes", index, x.data_ptr(), dtype, T, H, D, st[0], sh, pos.data_ptr(), pdt, ps, A,
                  ctypes.addressof(pairs), cos_sin.data_ptr(), P, r, D - r if rope_offset is None else int(rope_offset),
                  int(interleaved), int(inverse), out.data_ptr(), ost[0], osh)
        return out
    pos, pdt = _check_angles(index, cos_sin, positions, T, r)
    if T == 0 or H == 0:
        return out
    _call("nvfp4kv_rope", index, x.data_ptr(), dtype, T, H, D, st[0], sh, pos.data_ptr(), pdt,
          cos_sin.data_ptr(), P, r, D - r if rope_offset is None else int(rope_offset), int(interleaved),
          int(inverse), out.data_ptr(), ost[0], osh)
    return out


def write_nvfp4_rope_rotated(k_pe: torch.Tensor, rope_cache: torch.Tensor, slot_mapping: torch.Tensor,
                             positions: torch.Tensor, cos_sin: torch.Tensor, q_pe: torch.Tensor | None = None,
                             q_out: torch.Tensor | None = None, interleaved: bool = True,
                             axes=None) -> torch.Tensor | None:
    """The rope part of a step in one launch: k_pe [T, 64] bf16, rotated by its tokens' angles,
    into the rope side-pool at slot_mapping (as write_nvfp4_rope), and the queries' rope dims
    q_pe [T, H, 64] bf16 rotated into q_out (default: in place).  Returns q_out.  ``axes``: positions
    [axes, T], as in apply_rope."""
    _require_cuda(k_pe, "k_pe")
    index = k_pe.get_device()
    _require_on(index, rope_cache, "rope_cache")
    ks, (T, width) = k_pe.stride(), k_pe.shape if k_pe.dim() == 2 else (0, 0)
    if width < ROPE or k_pe.dtype is not torch.bfloat16 or ks[1] != 1:
        raise ValueError("k_pe must be bf16 [T, >=64] with a contiguous last dimension")
    if rope_cache.dtype is not torch.bfloat16:
        raise TypeError("rope_cache must be bf16")
    rows, rest = divmod(rope_cache.numel(), ROPE)
    if rest or not rope_cache.is_contiguous():
        raise ValueError("rope_cache must be contiguous rows of 64")
    _require_on(index, slot_mapping, "slot_mapping")
    slot = _vector(slot_mapping)
    if slot.shape[0] != T:
        raise ValueError(f"slot_mapping has {slot.shape[0]} entries for {T} tokens")
    sdt = _INDEX_DTYPES.get(slot.dtype)
    if sdt is None:
        raise TypeError("slot_mapping must be int64 or int32")
    if axes is None:
        pos, pdt = _check_angles(index, cos_sin, positions, T, ROPE)
    else:
        pos, pdt, ps, A, pairs = _check_axes(index, cos_sin, positions, T, ROPE, axes)
    H, qs, qos, q_ptr, qo_ptr = 0, (0, 0), (0, 0), 0, 0
    if q_pe is not None:
        _require_on(index, q_pe, "q_pe")
        shape, qs = q_pe.shape, q_pe.stride()
        if len(shape) != 3 or shape[0] != T or shape[2] != ROPE or qs[2] != 1 or q_pe.dtype is not torch.bfloat16:
            raise ValueError("q_pe must be bf16 [T, H, 64] with a contiguous last dimension")
        if q_out is None or q_out is q_pe:
            q_out, qos = q_pe, qs
        else:
            _require_on(index, q_out, "q_out")
            qos = q_out.stride()
            if q_out.shape != shape or qos[2] != 1 or q_out.dtype is not torch.bfloat16:
                raise ValueError("q_out must be bf16 of q_pe's shape with a contiguous last dimension")
        H = shape[1]
        if H:
            q_ptr, qo_ptr = q_pe.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q_pe")
    if T == 0:
        return q_out
    if axes is not None:
        _call("nvfp4kv_append_rope_rotated_axes", index, k_pe.data_ptr(), T, ks[0], rope_cache.data_ptr(),
              rows, slot.data_ptr(), sdt, pos.data_ptr(), pdt, ps, A, ctypes.addressof(pairs), cos_sin.data_ptr(),
              cos_sin.shape[0], int(interleaved), q_ptr, H, qs[0], qs[1], qo_ptr, qos[0], qos[1])
        return q_out
    _call("nvfp4kv_append_rope_rotated", index, k_pe.data_ptr(), T, ks[0], rope_cache.data_ptr(),
          rows, slot.data_ptr(), sdt, pos.data_ptr(), pdt, cos_sin.data_ptr(),
          cos_sin.shape[0], int(interleaved), q_ptr, H, qs[0], qs[1], qo_ptr, qos[0], qos[1])
    return q_out


# ------------------------------------------------------------------ chunk attention
def _window(window, sinks) -> tuple[int, int]:
    """A window and its sinks as C ints (what is longer than a sequence hides nothing)."""
    window, sinks = _whole(window, "window"), _whole(sinks, "sinks")
    if window < 0 or sinks < 0 or (sinks and not window):
        raise ValueError("window and sinks must be >= 0, and sinks need a window")
    return min(window, 0x7FFFFFFF), min(sinks, 0x7FFFFFFF)


def mla_prefill(query: torch.Tensor, kv_cache: torch.Tensor, workspace_buffer: torch.Tensor | None,
                kv_lora_rank: int, qk_rope_head_dim: int, block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor,
                seq_lens: torch.Tensor, max_q_len: int, max_seq_len: int, out: torch.Tensor | None = None,
                bmm1_scale: float = 1.0, bmm2_scale: float = 1.0, rope_cache: torch.Tensor | None = None,
                return_lse: bool = False, window: int = 0, sinks: int = 0):
    """Causal MLA attention of a ragged batch of new tokens over the paged pool, whose rows
    already hold them: chunked prefill, speculative steps and single tokens in one call.

    query [T, H, kv_lora_rank + qk_rope_head_dim] bf16: the new tokens of sequence b are
    cu_seqlens_q[b] .. cu_seqlens_q[b + 1], the last of its seq_lens[b] tokens; each sees the
    tokens up to itself.  kv_cache, block_tables, rope_cache and workspace_buffer as in
    mla_decode (dense).  max_q_len and max_seq_len bound the device-side lengths (a sequence past
    either is flagged in the device error word: it ends at max_seq_len tokens, and only its first
    max_q_len new tokens are computed); nothing synchronises the host.  Returns out
    [T, H, kv_lora_rank] bf16, with ``return_lse`` also lse [T, H] float32 (natural log; -inf for
    a row that sees no token, whose out is zeros).  Rows of new tokens past max_q_len, and rows
    from cu_seqlens_q[-1] on (the padding of a captured batch), are not written: they hold what
    was in ``out`` before, and anything where the call allocates it.

    ``window`` > 0: the query at position p sees only tokens t > p - window, and the first ``sinks``
    of its sequence.  What no new token sees is not read, and its pages may be gone (trim_pages).
    A call of many rows then takes the queries as they are: past 2^106 products can pass fp32's range."""
    try:      # (the whole host side of a call is about as long as a short batch on the device)
        index = query.get_device()
        together = index >= 0 and kv_cache.get_device() == block_tables.get_device() == cu_seqlens_q.get_device() \
            == seq_lens.get_device() == index and (rope_cache is None or rope_cache.get_device() == index)
    except AttributeError:
        together = False
    if not together:
        _require_cuda(query, "query")
        for name, t in (("kv_cache", kv_cache), ("block_tables", block_tables), ("cu_seqlens_q", cu_seqlens_q),
                        ("seq_lens", seq_lens), ("rope_cache", rope_cache)):
            _require_on(query.get_device(), t, name)
    if isinstance(bmm1_scale, torch.Tensor) or isinstance(bmm2_scale, torch.Tensor):
        raise TypeError("bmm1_scale / bmm2_scale must be Python floats (a device scalar would need a sync)")
    if window or sinks:
        window, sinks = _window(window, sinks)
    qs = query.stride()
    if query.dtype is not torch.bfloat16 or len(qs) != 3 or qs[2] != 1:
        raise ValueError("query must be bf16 [T, H, D] with a contiguous last dimension")
    T, H, D = query.shape
    if kv_lora_rank != LATENT or D != kv_lora_rank + qk_rope_head_dim:
        raise ValueError(f"query dim {D} must equal kv_lora_rank (512) + qk_rope_head_dim")
    pool = kv_cache.shape
    if pool[-1] != NV_BYTES or not kv_cache.is_contiguous():
        raise ValueError("kv_cache must be a contiguous pool of 288-byte rows")
    rows = kv_cache.numel() // NV_BYTES
    page_size = pool[-2] if len(pool) >= 3 else 64
    if not (block_tables.dtype is cu_seqlens_q.dtype is seq_lens.dtype is torch.int32):
        raise TypeError("block_tables, cu_seqlens_q and seq_lens must be int32")
    cu, sl = _vector(cu_seqlens_q), _vector(seq_lens)
    B, tables, ts = sl.shape[0], block_tables.shape, block_tables.stride()
    if len(tables) != 2 or tables[0] != B or (tables[1] > 1 and ts[1] != 1):
        raise ValueError("block_tables must be [B, width] with a contiguous last dimension")
    if cu.shape[0] != B + 1:
        raise ValueError("cu_seqlens_q must have one entry more than seq_lens")
    if tables[1] * page_size < max_seq_len:
        raise ValueError("block_tables too narrow for max_seq_len")
    if out is None:
        out = query.new_empty((T, H, LATENT))
        os = (H * LATENT, LATENT)
    else:
        os = out.stride()
        if out.get_device() != index or out.shape != (T, H, LATENT) or out.dtype is not torch.bfloat16 or os[2] != 1:
            raise ValueError("out must be bf16 [T, H, 512] on the device with a contiguous last dimension")
    rope = 0
    if rope_cache is not None:
        if rope_cache.dtype is not torch.bfloat16 or rope_cache.numel() != rows * ROPE or not rope_cache.is_contiguous():
            raise ValueError("rope_cache must be a contiguous bf16 [pool rows, 64] side-pool")
        rope = rope_cache.data_ptr()
    lse = query.new_empty((T, H), dtype=torch.float32) if return_lse else None
    if T > 0 and B > 0:
        key = ("prefill", B, T, H, max_q_len, max_seq_len, window, sinks, index)
        need = _ws_sizes.get(key)
        if need is None:
            n = ctypes.c_size_t(0)
            with _on_device(query.device):
                if window:
                    _lib.check(_lib.lib().nvfp4kv_mla_prefill_window_workspace_size(
                        B, T, H, int(max_q_len), int(max_seq_len), window, sinks, ctypes.byref(n)),
                        "nvfp4kv_mla_prefill_window_workspace_size")
                else:
                    _lib.check(_lib.lib().nvfp4kv_mla_prefill_workspace_size(B, T, H, int(max_q_len), int(max_seq_len),
                                                                             ctypes.byref(n)),
                               "nvfp4kv_mla_prefill_workspace_size")
            if len(_ws_sizes) >= 4096:      # a serving loop meets ever new shapes
                _ws_sizes.clear()
            need = _ws_sizes[key] = int(n.value)
        ws = workspace_buffer
        if ws is None or ws.get_device() != index or not ws.is_contiguous() or ws.data_ptr() % 256 \
                or ws.numel() * ws.element_size() < need:
            ws = _stream_buffer(index, "prefill_ws", need, torch.uint8)
        lse_ptr = 0 if lse is None else lse.data_ptr()
        if window:
            _call("nvfp4kv_mla_prefill_window", index, query.data_ptr(), qs[0], qs[1], kv_cache.data_ptr(), rows, rope,
                  block_tables.data_ptr(), ts[0], cu.data_ptr(), sl.data_ptr(), B, T, H, D, kv_lora_rank, page_size,
                  int(max_q_len), int(max_seq_len), window, sinks, bmm1_scale, bmm2_scale, out.data_ptr(), os[0], os[1],
                  lse_ptr, ws.data_ptr(), need)
        else:
            _call("nvfp4kv_mla_prefill", index, query.data_ptr(), qs[0], qs[1], kv_cache.data_ptr(), rows, rope,
                  block_tables.data_ptr(), ts[0], cu.data_ptr(), sl.data_ptr(), B, T, H, D, kv_lora_rank, page_size,
                  int(max_q_len), int(max_seq_len), bmm1_scale, bmm2_scale, out.data_ptr(), os[0], os[1], lse_ptr,
                  ws.data_ptr(), need)
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------ page upkeep
_MAX_CACHES = 8        # NVFP4KV_MAX_CACHES
_INT32 = torch.int32
_POINTERS, _SIZES = ctypes.c_void_p * _MAX_CACHES, ctypes.c_int64 * _MAX_CACHES


def _cache_list(caches):
    """(device pointers, bytes per page, their number, pages, page size, device) of pools [num_pages, page_size, ...]."""
    if not caches:
        raise ValueError("caches must name at least one pool")
    _require_cuda(caches[0], "caches")
    index = caches[0].get_device()
    pages, size = caches[0].shape[:2]
    n = len(caches)
    if n > _MAX_CACHES:
        raise ValueError(f"at most {_MAX_CACHES} caches in one call")
    ptrs, sizes = _POINTERS(), _SIZES()
    for k, c in enumerate(caches):
        if k:
            _require_on(index, c, "caches")
        shape = c.shape
        if len(shape) < 3 or shape[0] != pages or shape[1] != size or not c.is_contiguous():
            raise ValueError("caches must be contiguous [num_pages, page_size, ...] pools of one geometry")
        ptrs[k] = c.data_ptr()
        sizes[k] = c.nbytes // pages if pages else size
    return ptrs, sizes, n, pages, size, index


def _ints(index: int, *vectors) -> bool:
    """Whether all are contiguous int32 vectors on the device."""
    for t in vectors:
        if not isinstance(t, torch.Tensor) or t.dtype is not _INT32 or t.get_device() != index or t.dim() != 1 or not t.is_contiguous():
            return False
    return True


def _tables(index: int, tables: torch.Tensor, strides, *vectors) -> bool:
    """Whether ``tables`` is an int32 [slots, width] on the device with contiguous rows and the others
    are _ints."""
    return tables.dtype is _INT32 and len(strides) == 2 and strides[1] == 1 and _ints(index, *vectors)


def _check_int32(index: int, **tensors):
    """Says which of a call's tensors is not what it has to be."""
    for name, t in tensors.items():
        _require_on(index, t, name)
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32")
        if name.endswith("tables"):
            if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
                raise ValueError(f"{name} must be [slots, width] with a contiguous last dimension")
        elif t.dim() != 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous vector")


def _stream_buffer(index: int, name: str, n: int, dtype: torch.dtype) -> torch.Tensor:
    """A persistent buffer of the current stream, so that calls on two streams never share one.  A
    call that is being captured gets one from the graph's own pool: a persistent one may be
    replaced by a larger one while the graph lives."""
    if torch._C._cuda_isCurrentStreamCapturing():
        return torch.empty(n, dtype=dtype, device=torch.device("cuda", index))
    key = (name, index, _raw_stream(index))
    ws = _bufs.get(key)
    if ws is None or ws.numel() < n:
        ws = _bufs[key] = torch.empty(n, dtype=dtype, device=torch.device("cuda", index))
    return ws


class StepTables(NamedTuple):
    """What the kernels of a step take (extend_pages), for its n requests and num_tokens rows."""
    slot_mapping: torch.Tensor     # [num_tokens] int64: pool slot of each new token, -1 for padding
    positions: torch.Tensor        # [num_tokens] int32: its position, 0 for padding
    cu_seqlens_q: torch.Tensor     # [n + 1] int32: where each request's tokens begin
    seq_lens: torch.Tensor         # [n] int32: its length with them
    block_tables: torch.Tensor     # [n, width] int32: its table


def extend_pages(block_tables: torch.Tensor, seq_lens: torch.Tensor, slots: torch.Tensor, new_lens: torch.Tensor,
                 ref_counts: torch.Tensor, page_size: int, num_tokens: int,
                 lens: torch.Tensor | None = None) -> StepTables:
    """The tables of a step, built on the device: request k appends new_lens[k] tokens to the sequence
    in slots[k] of block_tables [num_slots, width] and seq_lens.  Every page that begins in them is
    the lowest free one (ref_counts 0 -> 1), in order of k; tables, lengths and counts change in
    place.  ``lens`` [n]: the sequences' lengths before the step where they are shorter than seq_lens
    (drafts that were not accepted are taken back, and their pages given back first).

    num_tokens: the step's rows, at least the new tokens; the rest is padding.  A request that cannot
    be extended is skipped, with no tokens, length 0 and an empty table, and flagged in the device
    error word: a bad or twice named slot, a bad length, more than the table's width, the free pages
    or num_tokens hold in order of k, or a first page that is missing or shared."""
    _require_cuda(block_tables, "block_tables")
    index, st = block_tables.get_device(), block_tables.stride()
    if not _tables(index, block_tables, st, seq_lens, slots, new_lens, ref_counts) or (lens is not None and not _ints(index, lens)):
        _check_int32(index, block_tables=block_tables, seq_lens=seq_lens, slots=slots, new_lens=new_lens, ref_counts=ref_counts,
                     **({} if lens is None else {"lens": lens}))
    n, (S, width), pages = slots.shape[0], block_tables.shape, ref_counts.shape[0]
    if seq_lens.shape[0] != S:
        raise ValueError("seq_lens must have one entry per row of block_tables")
    if new_lens.shape[0] != n or (lens is not None and lens.shape[0] != n):
        raise ValueError("new_lens and lens must have one entry per slot")
    if num_tokens < 0:
        raise ValueError("num_tokens must be >= 0")
    # (one allocation and one split: 5 us less than five; "unsafe" means that autograd does not know them as
    # views of one tensor)
    slot_words, tables, positions, out_lens, cu = torch.unsafe_split_with_sizes(
        block_tables.new_empty(n * width + 3 * num_tokens + 2 * n + 1), (2 * num_tokens, n * width, num_tokens, n, n + 1))
    slot_mapping = slot_words.view(torch.int64)
    need = 2 * n + S + pages       # nvfp4kv_extend_workspace_ints
    ws = _stream_buffer(index, "extend_ws", need, _INT32)
    _call("nvfp4kv_extend_pages", index, block_tables.data_ptr(), st[0], width, S, seq_lens.data_ptr(), slots.data_ptr(),
          new_lens.data_ptr(), 0 if lens is None else lens.data_ptr(), n, page_size, ref_counts.data_ptr(), pages,
          num_tokens, slot_mapping.data_ptr(), positions.data_ptr(), cu.data_ptr(), out_lens.data_ptr(), tables.data_ptr(),
          ws.data_ptr(), ws.numel())
    return StepTables(slot_mapping, positions, cu, out_lens, tables.view(n, width))


def trim_pages(block_tables: torch.Tensor, seq_lens: torch.Tensor, slots: torch.Tensor, ref_counts: torch.Tensor,
               page_size: int, window: int = 0, sinks: int = 0) -> None:
    """Gives back pages of the sequences in ``slots`` that no later step reads, in place: with
    ``window`` those behind the window of the next token, but for the first ``sinks`` tokens (their
    entries become -2), and those past the sequence's end (-1).  Where drafts may still be taken back, or
    cached tokens asked for again, give a window that is longer by their number."""
    _require_cuda(block_tables, "block_tables")
    index, st = block_tables.get_device(), block_tables.stride()
    if not _tables(index, block_tables, st, seq_lens, slots, ref_counts):
        _check_int32(index, block_tables=block_tables, seq_lens=seq_lens, slots=slots, ref_counts=ref_counts)
    S, width = block_tables.shape
    if seq_lens.numel() != S:
        raise ValueError("seq_lens must have one entry per row of block_tables")
    window, sinks = _window(window, sinks)
    _call("nvfp4kv_trim_pages", index, block_tables.data_ptr(), st[0], width, S, seq_lens.data_ptr(), slots.data_ptr(),
          slots.numel(), page_size, window, sinks, ref_counts.data_ptr(), ref_counts.numel())


def copy_pages(caches, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Pages src[k] -> dst[k] (int32) of every pool in ``caches`` ([num_pages, page_size, ...] each:
    latent rows, rope rows, indexer rows).  Negative ids skip the pair.  A page may not be a
    source and a destination, nor a destination twice."""
    ptrs, sizes, n, pages, _, index = _cache_list(caches)
    if not _ints(index, src, dst):
        _check_int32(index, src=src, dst=dst)
    if src.numel() != dst.numel():
        raise ValueError("src and dst must have the same length")
    _call("nvfp4kv_copy_pages", index, ctypes.addressof(ptrs), ctypes.addressof(sizes), n, pages, src.data_ptr(), dst.data_ptr(),
          src.shape[0])


def free_pages(block_tables: torch.Tensor, seq_lens: torch.Tensor, slots: torch.Tensor,
               ref_counts: torch.Tensor) -> None:
    """Empties the sequences in ``slots``: their pages lose one reference each (0 = free), their
    rows of block_tables [num_slots, width] become -1 and their seq_lens 0, in place."""
    _require_cuda(block_tables, "block_tables")
    index, st = block_tables.get_device(), block_tables.stride()
    if not _tables(index, block_tables, st, seq_lens, slots, ref_counts):
        _check_int32(index, block_tables=block_tables, seq_lens=seq_lens, slots=slots, ref_counts=ref_counts)
    S, width = block_tables.shape
    if seq_lens.numel() != S:
        raise ValueError("seq_lens must have one entry per row of block_tables")
    _call("nvfp4kv_free_pages", index, block_tables.data_ptr(), st[0], width, S, seq_lens.data_ptr(), slots.data_ptr(),
          slots.numel(), ref_counts.data_ptr(), ref_counts.numel())


def fork_pages(caches, block_tables: torch.Tensor, seq_lens: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               ref_counts: torch.Tensor) -> None:
    """Makes the empty slot dst[k] a copy of the sequence in slot src[k], for every k, in place:
    full pages are shared (one reference more each), the filled rows of a partly filled last
    page are copied in every pool of ``caches`` into the lowest free page (ref_counts == 0), in
    order of k.  Beams and samples that share a prompt; see free_pages for the way back."""
    ptrs, sizes, n, pages, size, index = _cache_list(caches)
    _require_on(index, block_tables, "block_tables")
    st = block_tables.stride()
    if not _tables(index, block_tables, st, seq_lens, src, dst, ref_counts):
        _check_int32(index, block_tables=block_tables, seq_lens=seq_lens, src=src, dst=dst, ref_counts=ref_counts)
    num = src.numel()
    if num != dst.numel():
        raise ValueError("src and dst must have the same length")
    S, width = block_tables.shape
    if seq_lens.numel() != S or ref_counts.numel() != pages:
        raise ValueError("seq_lens must have one entry per row of block_tables, ref_counts one per page")
    ws = _stream_buffer(index, "fork_ws", max(3 * num, 1024), _INT32)
    _call("nvfp4kv_fork_pages", index, ctypes.addressof(ptrs), ctypes.addressof(sizes), n, size, block_tables.data_ptr(),
          st[0], width, S, seq_lens.data_ptr(), src.data_ptr(), dst.data_ptr(), num, ref_counts.data_ptr(), pages, ws.data_ptr(),
          ws.numel())


def compact_pages(caches, block_tables: torch.Tensor, ref_counts: torch.Tensor, out_tables: torch.Tensor | None = None,
                  out_ref_counts: torch.Tensor | None = None) -> torch.Tensor:
    """Moves the pages in use (ref_counts > 0) to the front of every pool of ``caches``: the k-th of
    those past their number goes to the k-th free page before it.  The tables and counts that go
    with it are written to out_tables / out_ref_counts (default: in place; an engine whose
    running step still reads the old tables gives others).  Returns the number of pages in use,
    int32 [] on the device."""
    ptrs, sizes, n, pages, _, index = _cache_list(caches)
    _require_on(index, block_tables, "block_tables")
    ost = st = block_tables.stride()
    if not _tables(index, block_tables, st, ref_counts):
        _check_int32(index, block_tables=block_tables, ref_counts=ref_counts)
    if out_tables is None:
        out_tables = block_tables
    else:
        _check_int32(index, out_tables=out_tables)
        ost = out_tables.stride()
    if out_ref_counts is None:
        out_ref_counts = ref_counts
    else:
        _check_int32(index, out_ref_counts=out_ref_counts)
    if ref_counts.numel() != pages or out_ref_counts.numel() != pages or out_tables.shape != block_tables.shape:
        raise ValueError("ref_counts must have one entry per page, out_tables block_tables' shape")
    live = block_tables.new_empty(())
    need = _ws_sizes.get(("compact", pages))
    if need is None:
        n64 = ctypes.c_int64(0)
        _lib.check(_lib.lib().nvfp4kv_compact_workspace_ints(pages, ctypes.byref(n64)), "nvfp4kv_compact_workspace_ints")
        need = _ws_sizes["compact", pages] = int(n64.value)
    ws = _stream_buffer(index, "compact_ws", need, torch.int32)
    S, width = block_tables.shape
    _call("nvfp4kv_compact_pages", index, ctypes.addressof(ptrs), ctypes.addressof(sizes), n, block_tables.data_ptr(), st[0],
          width, S, ref_counts.data_ptr(), pages, out_tables.data_ptr(), ost[0], out_ref_counts.data_ptr(), live.data_ptr(),
          ws.data_ptr(), ws.numel())
    return live
