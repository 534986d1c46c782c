"""What the operators of caches in 8 bits refuse, without a GPU: the C entries' argument checks
(placeholder pointers that are never followed) and the Python checks."""

import pytest
import torch

from dropkv_b200 import _lib, load_rows_fp8, store_rows_fp8

P = 4096  # a placeholder device address


def _refused(rc, code, text):
    assert rc == code and text in _lib.load().dropkv_last_error().decode()


@pytest.mark.parametrize("change,code,text", [
    (dict(k=None), _lib.ERR_ARG, "NULL"), (dict(slots=None), _lib.ERR_ARG, "NULL"), (dict(kp=None), _lib.ERR_ARG, "pages and"),
    (dict(ks=None), _lib.ERR_ARG, "scales"), (dict(vs=P + 2), _lib.ERR_ARG, "scales"), (dict(dtype=3), _lib.ERR_ARG, "dtype"),
    (dict(B=-1), _lib.ERR_ARG, "sizes"), (dict(N=-1), _lib.ERR_ARG, "sizes"), (dict(D=0), _lib.ERR_ARG, "sizes"),
    (dict(H=0), _lib.ERR_ARG, "sizes"), (dict(block=0), _lib.ERR_ARG, "sizes"), (dict(k=P + 1), _lib.ERR_ARG, "aligned"),
    (dict(block=1025), _lib.ERR_UNSUPPORTED, "1024"), (dict(H=40000), _lib.ERR_UNSUPPORTED, "too many"),
    (dict(B=1 << 20, N=1 << 20), _lib.ERR_UNSUPPORTED, "too many"), (dict(N=(1 << 31) - 1), _lib.ERR_UNSUPPORTED, "too many"),
])
def test_store_rows_fp8_refuses(change, code, text):
    a = dict(k=P, v=P, slots=P, kp=P, vp=P, ks=P, vs=P, pages=4, block=16, dtype=2, B=1, H=2, N=3, D=64) | change
    s = (64, 64, 64)
    rc = _lib.load().dropkv_store_rows_fp8(a["k"], *s, a["v"], *s, a["slots"], a["kp"], *s, a["vp"], *s, a["ks"], 2, 1,
                                           a["vs"], 2, 1, a["pages"], a["block"], a["dtype"], a["B"], a["H"], a["N"],
                                           a["D"], None)
    _refused(rc, code, text)


@pytest.mark.parametrize("change,text", [
    (dict(slots=None), "NULL"), (dict(out=None), "NULL"), (dict(kp=None), "pages and"), (dict(ks=None), "scales"),
    (dict(dtype=-1), "dtype"), (dict(B=-1), "sizes"), (dict(D=0), "sizes"), (dict(block=0), "sizes"), (dict(out=P + 1), "aligned"),
])
def test_load_rows_fp8_refuses(change, text):
    a = dict(slots=P, kp=P, vp=P, ks=P, vs=P, pages=4, block=16, dtype=2, B=1, H=2, N=3, D=64, out=P) | change
    s = (64, 64, 64)
    rc = _lib.load().dropkv_load_rows_fp8(a["kp"], *s, a["vp"], *s, a["ks"], 2, 1, a["vs"], 2, 1, a["pages"], a["block"],
                                          a["slots"], a["dtype"], a["B"], a["H"], a["N"], a["D"], P, a["out"], None)
    _refused(rc, _lib.ERR_ARG, text)


class _Cuda(torch.Tensor):
    """A tensor that says it is on the current CUDA device."""

    def get_device(self):
        return 0


def _pool(pages=4, H=2, block=16, D=64):
    p = [torch.zeros(pages, H, block, D, dtype=torch.uint8).view(torch.float8_e4m3fn).as_subclass(_Cuda) for _ in "KV"]
    s = [torch.ones(pages, H).as_subclass(_Cuda) for _ in "KV"]
    return dict(K_pages=p[0], V_pages=p[1], K_scales=s[0], V_scales=s[1])


@pytest.fixture
def on_device_0(monkeypatch):
    from dropkv_b200 import paged
    monkeypatch.setattr(paged, "_current_device", lambda: 0)


@pytest.mark.parametrize("change,error,text", [
    (dict(K_pages=torch.zeros(4, 2, 16, 64)), TypeError, "float8"), (dict(V_pages=_pool(D=32)["V_pages"]), ValueError, "one shape"),
    (dict(K_scales=torch.ones(4, 2, dtype=torch.float64)), TypeError, "float32"), (dict(V_scales=torch.ones(4, 3)), ValueError, "pages, heads"),
    (dict(K=torch.zeros(1, 2, 3, 32), V=torch.zeros(1, 2, 3, 32)), ValueError, "fit"), (dict(V=torch.zeros(1, 2, 4, 64)), ValueError, "one shape"),
    (dict(K=torch.zeros(1, 2, 3, 64, dtype=torch.float64)), TypeError, "fp32"), (dict(slots=torch.zeros(1, 3, dtype=torch.int32)), TypeError, "slots"),
    (dict(slots=torch.zeros(1, 4, dtype=torch.int64)), ValueError, "slots"),
    (dict(K=torch.zeros(1, 2, 64, 3).transpose(2, 3)), ValueError, "contiguous"),
])
def test_store_rows_fp8_checks_its_tensors(change, error, text, on_device_0):
    x = torch.zeros(1, 2, 3, 64)
    a = dict(K=x, V=x, slots=torch.zeros(1, 3, dtype=torch.int64), **_pool()) | change
    with pytest.raises(error, match=text):
        store_rows_fp8(**{k: v.as_subclass(_Cuda) for k, v in a.items()})


def test_load_rows_fp8_checks_its_tensors(on_device_0):
    slots = torch.zeros(1, 3, dtype=torch.int64).as_subclass(_Cuda)
    with pytest.raises(TypeError, match="dtype"):
        load_rows_fp8(**_pool(), slots=slots, dtype=torch.int8)
    with pytest.raises(ValueError, match="slots"):
        load_rows_fp8(**_pool(), slots=slots[0])


def test_cpu_tensors_are_refused():
    x, slots = torch.zeros(1, 2, 3, 64), torch.zeros(1, 3, dtype=torch.int64)
    pool = {k: torch.Tensor(v).as_subclass(torch.Tensor) if v.dtype == torch.float32 else v.as_subclass(torch.Tensor)
            for k, v in _pool().items()}
    with pytest.raises(RuntimeError, match="CUDA"):
        store_rows_fp8(x, x, slots, **pool)
    with pytest.raises(RuntimeError, match="CUDA"):
        load_rows_fp8(**pool, slots=slots)
