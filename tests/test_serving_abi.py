"""CPU: the serving operators' C entry points are exported as declared and refuse bad calls before
any launch."""
import ctypes
import os
import re

import pytest
import torch

from conftest import ROOT
from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt

HEADER = os.path.join(ROOT, "include", "nvfp4kv_serving.h")


def refused(name, *args):
    lib = _lib.lib()
    rc = getattr(lib, name)(*args)
    return rc, lib.nvfp4kv_last_error().decode()


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(nvfp4kv_[a-z0-9_]+)\s*\(", text))
    assert names == set(_lib.SERVING_SIGNATURES)
    for n in names:
        assert hasattr(_lib.lib(), n), n


ROPE = dict(x=16, dtype=0, T=4, H=2, D=128, xt=256, xh=128, pos=16, pdt=0, cs=16, maxp=8, r=64, off=64, il=1, inv=0,
            out=4096, ot=256, oh=128, err=None, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(T=-1), "num_tokens"), (dict(dtype=5), "dtype"), (dict(pdt=4), "position dtype"), (dict(H=0), "num_heads"),
    (dict(r=63), "rotary_dim"), (dict(off=65), "rotary_dim"), (dict(off=-2), "rotary_dim"), (dict(maxp=0), "cos_sin"),
    (dict(x=None), "null"), (dict(out=None), "null"), (dict(x=17), "aligned"), (dict(out=16, oh=64), "in place"),
])
def test_rope_refuses(change, word):
    rc, msg = refused("nvfp4kv_rope", *(ROPE | change).values())
    assert rc == _lib.EINVAL and word in msg


def test_rope_of_no_tokens_is_a_no_op():
    assert refused("nvfp4kv_rope", *(ROPE | dict(T=0, x=None)).values())[0] == _lib.OK


WRITE = dict(k=16, T=4, ks=64, pool=4096, rows=64, slots=16, sdt=0, pos=16, pdt=0, cs=16, maxp=8, il=1, q=32, H=2,
             qt=128, qh=64, qo=64, qot=128, qoh=64, err=None, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(T=-1), "num_tokens"), (dict(sdt=2), "int64 or int32"), (dict(pdt=2), "int64 or int32"), (dict(k=None), "null"),
    (dict(qo=None), "null"), (dict(ks=63), "k_stride"), (dict(rows=0), "empty"), (dict(maxp=0), "empty"),
    (dict(H=0), "num_heads"), (dict(pool=8), "aligned"), (dict(cs=4), "aligned"), (dict(qo=32, qoh=32), "in place"),
])
def test_rotated_rows_refuse(change, word):
    rc, msg = refused("nvfp4kv_append_rope_rotated", *(WRITE | change).values())
    assert rc == _lib.EINVAL and word in msg


PREFILL = dict(q=16, qt=1152, qh=576, pool=4096, rows=128, rope=None, tab=16, ts=2, cu=16, seq=16, B=1, T=2, H=2, D=576,
               rank=512, page=64, mq=2, ms=128, s1=1.0, s2=1.0, out=4096, ot=1024, oh=512, lse=None, ws=None, wb=0,
               err=None, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(B=-1), "batch"), (dict(T=-1), "total_q"), (dict(H=0), "num_heads"), (dict(rank=256), "kv_lora_rank"),
    (dict(D=500), "head_dim_qk"), (dict(D=512, rope=16), "head_dim_qk"), (dict(page=48), "page_size"),
    (dict(page=8192), "page_size"), (dict(q=None), "null"), (dict(cu=None), "null"), (dict(rows=100), "pool_rows"),
    (dict(pool=4104), "aligned"), (dict(qh=100), "multiples"), (dict(rope=24), "aligned"), (dict(out=4100), "aligned"),
    (dict(oh=100), "multiples"), (dict(ms=-1), "max_seq_len"), (dict(H=1 << 30, mq=8), "too many"),
])
def test_prefill_refuses(change, word):
    rc, msg = refused("nvfp4kv_mla_prefill", *(PREFILL | change).values())
    assert rc == _lib.EINVAL and word in msg


def test_prefill_of_nothing_is_a_no_op():
    assert refused("nvfp4kv_mla_prefill", *(PREFILL | dict(T=0, q=None)).values())[0] == _lib.OK
    assert refused("nvfp4kv_mla_prefill", *(PREFILL | dict(B=0, seq=None)).values())[0] == _lib.OK


def test_prefill_workspace_size_checks():
    n = ctypes.c_size_t(7)
    assert refused("nvfp4kv_mla_prefill_workspace_size", 2, 3, 0, 1, 64, ctypes.byref(n))[0] == _lib.EINVAL
    assert refused("nvfp4kv_mla_prefill_workspace_size", 2, 3, 4, 1, 64, None)[0] == _lib.EINVAL


def test_page_calls_refuse():
    ptrs, sizes = (ctypes.c_void_p * 2)(4096, 8192), (ctypes.c_int64 * 2)(64 * 288, 64 * 72)
    null = (ctypes.c_void_p * 2)(4096, None)
    copy = lambda c=ptrs, b=sizes, n=2, pages=4, src=16, dst=16, k=3: refused("nvfp4kv_copy_pages", c, b, n, pages, src, dst, k, None, None)  # noqa: E731
    for (rc, msg), word in [(copy(k=-1), "num_pairs"), (copy(n=9), "caches"), (copy(c=None), "null"), (copy(c=null), "null"),
                            (copy(src=None), "null"), (copy(pages=0), "num_pages"),
                            (copy(b=(ctypes.c_int64 * 2)(0, 72)), "page_bytes")]:
        assert rc == _lib.EINVAL and word in msg, msg
    assert copy(k=0)[0] == _lib.OK
    free = dict(t=16, ts=4, w=4, slots=3, seq=16, ids=16, n=2, refs=16, pages=8, err=None, st=None)
    for change, word in [(dict(n=-1), "num"), (dict(ids=None), "null"), (dict(refs=None), "null"), (dict(ts=3), "table"),
                         (dict(w=0), "table"), (dict(pages=0), "num_pages")]:
        rc, msg = refused("nvfp4kv_free_pages", *(free | change).values())
        assert rc == _lib.EINVAL and word in msg, msg
    fork = dict(c=ptrs, b=sizes, n=2, page=64, t=16, ts=4, w=4, slots=3, seq=16, src=16, dst=16, k=2, refs=16, pages=8,
                ws=16, wi=6, err=None, st=None)
    for change, word in [(dict(k=-1), "num"), (dict(page=0), "page_size"), (dict(page=7), "page_bytes"), (dict(src=None), "null"),
                         (dict(seq=None), "null"), (dict(t=None), "null")]:
        rc, msg = refused("nvfp4kv_fork_pages", *(fork | change).values())
        assert rc == _lib.EINVAL and word in msg, msg
    assert refused("nvfp4kv_fork_pages", *(fork | dict(wi=5)).values())[0] == _lib.EWORKSPACE
    n = ctypes.c_int64(0)
    assert refused("nvfp4kv_compact_workspace_ints", 8, ctypes.byref(n))[0] == _lib.OK and n.value > 0
    compact = dict(c=ptrs, b=sizes, n=2, t=16, ts=4, w=4, slots=3, refs=16, pages=8, ot=16, ots=4, orf=16, live=16, ws=16,
                   wi=n.value, err=None, st=None)
    for change, word in [(dict(ot=None), "output"), (dict(ots=3), "output"), (dict(live=None), "output"), (dict(refs=None), "null")]:
        rc, msg = refused("nvfp4kv_compact_pages", *(compact | change).values())
        assert rc == _lib.EINVAL and word in msg, msg
    assert refused("nvfp4kv_compact_pages", *(compact | dict(wi=n.value - 1)).values())[0] == _lib.EWORKSPACE


def test_python_entries_refuse_cpu_tensors_and_bad_tables():
    x = torch.zeros(2, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        rt.apply_rope(x, torch.zeros(2, dtype=torch.int32), torch.zeros(4, 64))
    with pytest.raises(ValueError, match="CUDA"):
        rt.copy_pages([torch.zeros(2, 2, 8)], torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="at least one"):
        rt.copy_pages([], None, None)
    with pytest.raises(ValueError, match="rotary_dim"):
        rt.rope_cos_sin(8, 63)


def test_tensors_of_another_device_are_refused():
    class Elsewhere(torch.Tensor):
        """A CPU tensor that says it is on the second GPU."""
        is_cuda = True

        def get_device(self):
            return 1

    t = torch.zeros(4).as_subclass(Elsewhere)
    rt._require_on(1, t, "t")
    with pytest.raises(ValueError, match="t must be on cuda:0"):
        rt._require_on(0, t, "t")
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        rt._require_on(0, torch.zeros(4), "t")
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        rt._require_on(0, None, "t")
