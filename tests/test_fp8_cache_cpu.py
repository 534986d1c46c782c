"""What the operators of caches in 8 bits refuse, without a GPU: the C entries' argument checks
(placeholder pointers that are never followed) and the Python checks."""

import pytest
import torch

from dropkv_b200 import _lib, attention_fp8, load_rows_fp8, store_rows_fp8, verify_draft

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


def _attention(change):
    a = dict(q=P, kp=P, vp=P, ks=P, vs=P, st=(2048, 1024, 64), pages=4, block=16, table=P, max_blocks=3, lens=P, mask=None,
             window=0, sinks=0, dtype=2, B=1, Hq=4, Hkv=2, T=5, D=64, scale=0.1, out=P, ws=None, have=0) | change
    return _lib.load().dropkv_attention_fp8(
        a["q"], 64, 64, 64, 1, a["kp"], *a["st"], a["vp"], *a["st"], a["ks"], 2, 1, a["vs"], 2, 1, a["pages"], a["block"],
        a["table"], a["max_blocks"], a["lens"], a["mask"], 0, 5, 1, a["window"], a["sinks"], a["dtype"], a["B"], a["Hq"],
        a["Hkv"], a["T"], a["D"], a["scale"], a["out"], a["ws"], a["have"], None)


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), _lib.ERR_ARG, "NULL"), (dict(lens=None), _lib.ERR_ARG, "NULL"), (dict(out=None), _lib.ERR_ARG, "NULL"),
    (dict(table=None), _lib.ERR_ARG, "table"), (dict(kp=None), _lib.ERR_ARG, "pages and"), (dict(vs=None), _lib.ERR_ARG, "scales"),
    (dict(dtype=0), _lib.ERR_UNSUPPORTED, "bf16 or fp16"), (dict(D=96), _lib.ERR_UNSUPPORTED, "64 or 128"),
    (dict(block=24), _lib.ERR_UNSUPPORTED, "power of two"), (dict(block=4), _lib.ERR_UNSUPPORTED, "power of two"),
    (dict(block=2048), _lib.ERR_UNSUPPORTED, "power of two"), (dict(max_blocks=1 << 27), _lib.ERR_UNSUPPORTED, "too long"),
    (dict(max_blocks=-1), _lib.ERR_UNSUPPORTED, "too long"), (dict(Hq=258), _lib.ERR_UNSUPPORTED, "128 query heads"),
    (dict(Hq=5), _lib.ERR_ARG, "sizes"), (dict(T=0), _lib.ERR_ARG, "sizes"), (dict(B=40000), _lib.ERR_ARG, "sizes"),
    (dict(T=257, mask=P), _lib.ERR_UNSUPPORTED, "256 nodes"), (dict(window=-1), _lib.ERR_ARG, "negative"),
    (dict(sinks=-1), _lib.ERR_ARG, "negative"), (dict(window=4, mask=P), _lib.ERR_ARG, "whole tree"),
    (dict(kp=P + 8), _lib.ERR_ARG, "16-byte"), (dict(st=(2048, 1024, 72)), _lib.ERR_ARG, "16-byte"),
    (dict(st=(2048, 1024, 48)), _lib.ERR_ARG, "strides"), (dict(q=P + 1), _lib.ERR_ARG, "aligned"), (dict(out=P + 2), _lib.ERR_ARG, "aligned"),
    (dict(scale=0.0), _lib.ERR_ARG, "scale"), (dict(scale=float("nan")), _lib.ERR_ARG, "scale"),
    (dict(scale=float("inf")), _lib.ERR_ARG, "scale"), (dict(scale=3e38), _lib.ERR_ARG, "scale"),
    (dict(), _lib.ERR_WORKSPACE, "workspace"), (dict(T=40), _lib.ERR_WORKSPACE, "workspace"),
])
def test_attention_fp8_refuses(change, code, text):
    _refused(_attention(change), code, text)


def test_attention_workspaces():
    size = _lib.load().dropkv_attention_fp8_workspace_size
    assert size(1, 6, 4, 5, 128, 100) == 0 and size(1, 8, 4, 5, 96, 100) == 0 and size(1, 258, 2, 1, 128, 100) == 0
    # the partials of two pieces a CTA; more rows than a tile's add what their queries take in 8 bits
    assert 0 < size(1, 32, 8, 1, 128, 1000) < size(1, 32, 8, 64, 128, 1000) < size(1, 32, 8, 4096, 128, 1000)


@pytest.mark.parametrize("change,error,text", [
    (dict(Q=torch.zeros(1, 4, 3, 64)), TypeError, "bf16 or fp16"), (dict(Q=torch.zeros(4, 3, 64)), ValueError, "expected Q"),
    (dict(Q=torch.zeros(1, 4, 3, 128, dtype=torch.bfloat16)), ValueError, "mismatch"),
    (dict(Q=torch.zeros(1, 5, 3, 64, dtype=torch.bfloat16)), ValueError, "mismatch"),
    (dict(cache_lens=torch.zeros(1, dtype=torch.int64)), TypeError, "cache_lens"), (dict(cache_lens=torch.zeros(2, dtype=torch.int32)), ValueError, "cache_lens"),
    (dict(block_table=torch.zeros(4, dtype=torch.int32)), ValueError, "block_table"), (dict(block_table=torch.zeros(2, 4, dtype=torch.int32)), ValueError, "block_table"),
    (dict(tree_mask=torch.ones(3, 3)), TypeError, "bool"), (dict(tree_mask=torch.ones(3, 4, dtype=torch.bool)), ValueError, "tree_mask"),
    (dict(K_pages=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)), TypeError, "float8"),
])
def test_attention_fp8_checks_its_tensors(change, error, text, on_device_0):
    a = dict(Q=torch.zeros(1, 4, 3, 64, dtype=torch.bfloat16), **_pool(), cache_lens=torch.zeros(1, dtype=torch.int32),
             block_table=torch.zeros(1, 4, dtype=torch.int32)) | change
    with pytest.raises(error, match=text):
        attention_fp8(**{k: v.as_subclass(_Cuda) for k, v in a.items()})


@pytest.mark.parametrize("window", [0, -3])
def test_attention_fp8_refuses_empty_windows(window, on_device_0):
    a = dict(Q=torch.zeros(1, 4, 3, 64, dtype=torch.bfloat16), **_pool(), cache_lens=torch.zeros(1, dtype=torch.int32),
             block_table=torch.zeros(1, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="window"):
        attention_fp8(**{k: v.as_subclass(_Cuda) for k, v in a.items()}, window=window)


class _OnDevice(torch.Tensor):
    """A tensor that says it is on CUDA device 3."""

    def get_device(self):
        return 3


@pytest.mark.parametrize("op,arguments", [
    (store_rows_fp8, dict(slots=None, K=None, V=None, K_pages=None, V_pages=None, K_scales=None, V_scales=None)),
    (load_rows_fp8, dict(dtype=torch.float16, K_pages=None, V_pages=None, K_scales=None, V_scales=None, slots=None)),
    (attention_fp8, dict(scale=0.1, tree_mask="none", Q=None, K_pages=None, V_pages=None, K_scales=None, V_scales=None,
                         cache_lens=None, block_table=None)),
    (verify_draft, dict(temperature=0.5, draft_logits="none", target_logits=None, tokens=None, uniforms=None)),
])
def test_calls_enter_their_tensors_device(op, arguments, monkeypatch):
    from dropkv_b200 import paged
    entered = []

    class Entered(Exception):
        pass

    class Device:
        def __init__(self, index):
            entered.append(index)

        def __enter__(self):
            raise Entered

        def __exit__(self, *a):
            return False

    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    x = torch.zeros(2).as_subclass(_OnDevice)
    arguments = {k: x if v is None else None if v == "none" else v for k, v in arguments.items()}
    with pytest.raises(Entered):
        op(**arguments)
    assert entered == [3]


def test_arguments_in_one_array():
    """The entries that take them so refuse what the plain ones do, and integers that no argument holds."""
    pool = (P, 64, 64, 64, P, 64, 64, 64, P, 2, 1, P, 2, 1)
    pack, call = _lib.words("dropkv_load_rows_fp8")
    _refused(call(pack(*pool, 4, 16, 0, 2, 1, 2, 3, 64, P, P, 0)), _lib.ERR_ARG, "NULL")
    _refused(call(pack(*pool, 4, 16, P, 2, 1, 2, 3, 64, P, P + 1, 0)), _lib.ERR_ARG, "aligned")
    for at in (14, 15, 17, 18, 20, 21):
        args = [*pool, 4, 16, P, 2, 1, 2, 3, 64, P, P, 0]
        args[at] = (1 << 32) + args[at]
        _refused(call(pack(*args)), _lib.ERR_ARG, "out of range")
    pack, call = _lib.words("dropkv_verify_draft")
    for tau, text in ((0.0, "temperature"), (float("nan"), "temperature"), (0.5, "workspace")):
        rc = call(pack(P, 400, 100, 0, 0, 0, 2, P, P, 2, 3, 100, tau, P, P, P, 0, 0, 0))
        assert rc != _lib.OK and text in _lib.load().dropkv_last_error().decode()
    for name in _lib.IN_WORDS:
        assert getattr(_lib.load(), name + "_words")(None) == _lib.ERR_ARG
