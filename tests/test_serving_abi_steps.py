"""CPU: the C entry points of a step's tables, of rotary positions with several axes and of the windowed
chunk attention refuse bad calls before any launch, and the host-side pieces of their Python entries."""
import ctypes

import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import _lib
from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt


def refused(name, *args):
    lib = _lib.lib()
    rc = getattr(lib, name)(*args)
    return rc, lib.nvfp4kv_last_error().decode()


def pairs(*axes):
    return (ctypes.c_uint8 * len(axes))(*axes)


ROPE = dict(x=16, dtype=0, T=4, H=2, D=128, xt=256, xh=128, pos=16, pdt=0, ps=4, A=3, ax=pairs(*[0, 1, 2, 2] * 8), cs=16, maxp=8,
            r=64, off=64, il=1, inv=0, out=4096, ot=256, oh=128, err=None, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(A=0), "num_axes"), (dict(A=5), "num_axes"), (dict(A=-1), "num_axes"), (dict(ax=None), "null"), (dict(A=2), "axis 2 of 2"),
    (dict(D=600, r=258, off=0), "at most 256"), (dict(T=-1), "num_tokens"), (dict(dtype=5), "dtype"), (dict(pdt=4), "position dtype"),
    (dict(r=63), "rotary_dim"), (dict(x=None), "null"), (dict(pos=None), "null"), (dict(x=17), "aligned"), (dict(out=16, oh=64), "in place"),
])
def test_rope_axes_refuses(change, word):
    rc, msg = refused("nvfp4kv_rope_axes", *(ROPE | change).values())
    assert rc == _lib.EINVAL and word in msg and msg.startswith("nvfp4kv_rope_axes")


WRITE = dict(k=16, T=4, ks=64, pool=4096, rows=64, slots=16, sdt=0, pos=16, pdt=0, ps=4, A=3, ax=pairs(*[0, 1, 2, 2] * 8), cs=16,
             maxp=8, il=1, q=32, H=2, qt=128, qh=64, qo=64, qot=128, qoh=64, err=None, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(A=0), "num_axes"), (dict(A=5), "num_axes"), (dict(ax=None), "null"), (dict(ax=pairs(*[3] * 32)), "axis 3 of 3"),
    (dict(T=-1), "num_tokens"), (dict(k=None), "null"), (dict(rows=0), "empty"), (dict(cs=4), "aligned"), (dict(qo=32, qoh=32), "in place"),
])
def test_rotated_rows_of_several_axes_refuse(change, word):
    rc, msg = refused("nvfp4kv_append_rope_rotated_axes", *(WRITE | change).values())
    assert rc == _lib.EINVAL and word in msg


PREFILL = dict(q=16, qt=1152, qh=576, pool=4096, rows=128, rope=None, tab=16, ts=2, cu=16, seq=16, B=1, T=2, H=2, D=576,
               rank=512, page=64, mq=2, ms=128, win=40, sinks=4, s1=1.0, s2=1.0, out=4096, ot=1024, oh=512, lse=None, ws=None, wb=0,
               err=None, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(win=0), "window"), (dict(win=-3), "window"), (dict(sinks=-1), "window"), (dict(B=-1), "batch"), (dict(H=0), "num_heads"),
    (dict(rank=256), "kv_lora_rank"), (dict(D=512, rope=16), "head_dim_qk"), (dict(page=48), "page_size"), (dict(cu=None), "null"),
    (dict(rows=100), "pool_rows"), (dict(pool=4104), "aligned"), (dict(oh=100), "multiples"), (dict(ms=-1), "max_seq_len"),
    (dict(H=1 << 30, mq=8), "too many"),
])
def test_windowed_prefill_refuses(change, word):
    rc, msg = refused("nvfp4kv_mla_prefill_window", *(PREFILL | change).values())
    assert rc == _lib.EINVAL and word in msg


def test_nothing_to_do_is_a_no_op():
    assert refused("nvfp4kv_mla_prefill_window", *(PREFILL | dict(T=0, q=None)).values())[0] == _lib.OK
    assert refused("nvfp4kv_rope_axes", *(ROPE | dict(T=0, x=None)).values())[0] == _lib.OK
    assert refused("nvfp4kv_trim_pages", *(TRIM | dict(num=0, slots=None)).values())[0] == _lib.OK


def size(*a):
    out = ctypes.c_size_t(0)
    rc, msg = refused("nvfp4kv_mla_prefill_window_workspace_size", *a, ctypes.byref(out))
    return rc, out.value, msg


def test_window_workspace():
    assert size(1, 2, 2, 2, 128, 0, 0)[0] == _lib.EINVAL and size(1, 2, 2, 2, 128, 4, -1)[0] == _lib.EINVAL
    assert size(0, 0, 2, 2, 128, 4, 0) [:2] == (_lib.OK, 0)
    whole = ctypes.c_size_t(0)
    assert refused("nvfp4kv_mla_prefill_workspace_size", 8, 4096, 64, 2048, 300000, ctypes.byref(whole))[0] == _lib.OK
    rc, need, _ = size(8, 4096, 64, 2048, 300000, 4096, 64)
    assert rc == _lib.OK and 0 < need < whole.value          # the windows' images, not the contexts'
    # a window that hides nothing is none
    assert size(8, 4096, 64, 2048, 300000, 299990, 10)[1] == whole.value == size(8, 4096, 64, 2048, 300000, 2 ** 31 - 1, 2 ** 31 - 1)[1]


EXTEND = dict(tab=16, ts=8, width=8, S=4, seq=16, slots=16, new=16, lens=None, num=2, page=16, refs=16, pages=9, T=4, sm=16, pos=16, cu=16,
              ol=16, ot=16, ws=16, wi=100, err=None, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(num=-1), "num"), (dict(T=-1), "num_tokens"), (dict(page=0), "page_size"), (dict(tab=None), "null"), (dict(refs=None), "null"),
    (dict(width=0), "table shape"), (dict(ts=7), "table shape"), (dict(S=0), "table shape"), (dict(pages=0), "num_pages"),
    (dict(width=1 << 20, ts=1 << 20, page=4096), "2^31"), (dict(T=1 << 31), "2^31"), (dict(cu=None), "null"), (dict(sm=None), "null"),
    (dict(pos=None), "null"), (dict(new=None), "null"), (dict(slots=None), "null"), (dict(ol=None), "null"), (dict(ot=None), "null"),
])
def test_extend_refuses(change, word):
    rc, msg = refused("nvfp4kv_extend_pages", *(EXTEND | change).values())
    assert rc == _lib.EINVAL and word in msg


def test_extend_workspace():
    ints = ctypes.c_int64(0)
    assert refused("nvfp4kv_extend_workspace_ints", 2, 4, 9, ctypes.byref(ints))[0] == _lib.OK
    assert refused("nvfp4kv_extend_pages", *(EXTEND | dict(wi=ints.value - 1)).values())[0] == _lib.EWORKSPACE
    assert refused("nvfp4kv_extend_pages", *(EXTEND | dict(ws=None)).values())[0] == _lib.EWORKSPACE
    assert refused("nvfp4kv_extend_workspace_ints", 2, 4, 9, None)[0] == _lib.EINVAL
    assert refused("nvfp4kv_extend_workspace_ints", -1, 4, 9, ctypes.byref(ints))[0] == _lib.EINVAL


TRIM = dict(tab=16, ts=8, width=8, S=4, seq=16, slots=16, num=2, page=16, win=4, sinks=0, refs=16, pages=9, err=None, st=None)


@pytest.mark.parametrize("change,word", [
    (dict(num=-1), "num"), (dict(page=0), "page_size"), (dict(win=-1), "window"), (dict(sinks=-1), "window"), (dict(slots=None), "null"),
    (dict(seq=None), "null"), (dict(refs=None), "null"), (dict(width=9), "table shape"),
])
def test_trim_refuses(change, word):
    rc, msg = refused("nvfp4kv_trim_pages", *(TRIM | change).values())
    assert rc == _lib.EINVAL and word in msg


def test_rope_axes():
    assert rt.rope_axes((2, 1, 1), 8) == (0, 0, 1, 2)
    assert rt.rope_axes((3, 1, 2), 12, dealt=True) == (0, 1, 2, 0, 2, 0)
    assert rt.rope_axes((32,)) == (0,) * 32 and rt.rope_axes((0, 32)) == (1,) * 32
    for bad in ((), (1, 2), (8,) * 5, (33, -1)):
        with pytest.raises(ValueError, match="sections"):
            rt.rope_axes(bad)


def test_cpu_tensors_are_refused():
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="CUDA"):
        rt.extend_pages(i(0).view(1, 1), i(0), i(0), i(1), i(0), 16, 1)
    with pytest.raises(ValueError, match="CUDA"):
        rt.trim_pages(i(0).view(1, 1), i(0), i(0), i(0), 16)


# ------------------------------------------------------------------ packed calls
def packed_refused(name, args):
    number, num, pack = _lib.packed(name)
    words = [0 if a is None else ctypes.addressof(a) if isinstance(a, ctypes.Array) else a for a in args]
    lib = _lib.lib()
    return lib.nvfp4kv_call_packed(number, num, pack(*words)), lib.nvfp4kv_last_error().decode()


def test_every_entry_with_a_stream_has_a_packed_form():
    numbers = set()
    for name, (_, types) in _lib.SERVING_SIGNATURES.items():
        if "_workspace_" in name or "packed" in name:
            with pytest.raises(_lib.Nvfp4kvError, match="no entry"):
                _lib.packed(name)
        else:
            number, num, _ = _lib.packed(name)
            assert num == len(types)
            numbers.add(number)
    assert numbers == set(range(len(numbers)))


@pytest.mark.parametrize("name,case,change", [
    ("nvfp4kv_rope_axes", ROPE, dict(A=2)), ("nvfp4kv_rope_axes", ROPE, dict(D=600, r=258, off=0)), ("nvfp4kv_rope_axes", ROPE, dict(T=0)),
    ("nvfp4kv_rope_axes", ROPE, dict(T=-1)), ("nvfp4kv_append_rope_rotated_axes", WRITE, dict(qo=32, qoh=32)),
    ("nvfp4kv_append_rope_rotated_axes", WRITE, dict(T=0)), ("nvfp4kv_mla_prefill_window", PREFILL, dict(rows=100)),
    ("nvfp4kv_mla_prefill_window", PREFILL, dict(rows=(1 << 40) + 1)), ("nvfp4kv_mla_prefill_window", PREFILL, dict(T=0)),
    ("nvfp4kv_extend_pages", EXTEND, dict(ws=None)), ("nvfp4kv_trim_pages", TRIM, dict(width=9)), ("nvfp4kv_trim_pages", TRIM, dict(num=0)),
])
def test_a_packed_call_is_the_call(name, case, change):
    args = list((case | change).values())
    want = refused(name, *args)
    got = packed_refused(name, args)
    assert got[0] == want[0] and (got[0] == _lib.OK or got == want)


def test_packed_calls_refuse():
    lib = _lib.lib()
    number, num, pack = _lib.packed("nvfp4kv_trim_pages")
    for change in (dict(num=1 << 31), dict(win=-(1 << 31) - 1), dict(page=1 << 40)):      # (a foreign call would cut them off)
        rc, msg = packed_refused("nvfp4kv_trim_pages", (TRIM | change).values())
        assert rc == _lib.EINVAL and "does not fit" in msg and str(list(TRIM).index(next(iter(change)))) in msg
    for entry, n, words in ((-1, num, b""), (1000, num, b""), (number, num - 1, b""), (number, num, None)):
        assert lib.nvfp4kv_call_packed(entry, n, words) == _lib.EINVAL
    out = ctypes.c_int(0)
    assert lib.nvfp4kv_packed_entry(None, ctypes.byref(out), ctypes.byref(out)) == _lib.EINVAL
    assert lib.nvfp4kv_packed_entry(b"nvfp4kv_append", ctypes.byref(out), ctypes.byref(out)) == _lib.EINVAL
    assert lib.nvfp4kv_packed_entry(b"nvfp4kv_rope", None, ctypes.byref(out)) == _lib.EINVAL


def test_an_argument_of_another_type_is_a_type_error(monkeypatch):
    monkeypatch.setitem(rt._bufs, ("err", 0), torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(rt, "_raw_stream", lambda index: 0)
    for bad in (1.5, None, "16", 1 << 70):
        with pytest.raises(TypeError, match="nvfp4kv_trim_pages"):
            rt._call("nvfp4kv_trim_pages", 0, *list((TRIM | dict(page=bad)).values())[:-2])
