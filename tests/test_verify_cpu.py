"""What ``verify_draft`` refuses, without a GPU: the C entry's argument checks (placeholder pointers that are
never followed) and the Python checks."""

import pytest
import torch

from dropkv_b200 import _lib, verify_draft

P = 4096  # a placeholder device address


@pytest.mark.parametrize("change,code,text", [
    (dict(target=None), _lib.ERR_ARG, "NULL"), (dict(tokens=None), _lib.ERR_ARG, "NULL"), (dict(u=None), _lib.ERR_ARG, "NULL"),
    (dict(acc=None), _lib.ERR_ARG, "NULL"), (dict(prob=None), _lib.ERR_ARG, "NULL"), (dict(dtype=9), _lib.ERR_ARG, "dtype"),
    (dict(B=-1), _lib.ERR_ARG, "sizes"), (dict(T=-1), _lib.ERR_ARG, "sizes"), (dict(V=0), _lib.ERR_ARG, "sizes"),
    (dict(T=257), _lib.ERR_UNSUPPORTED, "256 drafted"), (dict(V=(1 << 21) + 1), _lib.ERR_UNSUPPORTED, "vocabularies"),
    (dict(target=P + 1), _lib.ERR_ARG, "aligned"), (dict(draft=P + 1), _lib.ERR_ARG, "aligned"), (dict(tau=0.0), _lib.ERR_ARG, "temperature"),
    (dict(tau=-1.0), _lib.ERR_ARG, "temperature"), (dict(tau=1e-7), _lib.ERR_ARG, "temperature"), (dict(tau=1e7), _lib.ERR_ARG, "temperature"),
    (dict(tau=float("nan")), _lib.ERR_ARG, "temperature"), (dict(), _lib.ERR_WORKSPACE, "workspace"),
])
def test_verify_draft_refuses(change, code, text):
    a = dict(target=P, draft=P, dtype=2, tokens=P, u=P, B=2, T=3, V=100, tau=1.0, acc=P, nxt=P, prob=P) | change
    lib = _lib.load()
    rc = lib.dropkv_verify_draft(a["target"], 400, 100, a["draft"], 300, 100, a["dtype"], a["tokens"], a["u"], a["B"], a["T"],
                                 a["V"], a["tau"], a["acc"], a["nxt"], a["prob"], None, 0, None)
    assert rc == code and text in lib.dropkv_last_error().decode()


def test_workspaces_of_invalid_problems_are_empty():
    size = _lib.load().dropkv_verify_draft_workspace_size
    assert size(0, 3, 100, 1) == 0 and size(1, 300, 100, 1) == 0 and size(1, 3, 0, 1) == 0 and size(1, 3, 100, 1) > 0


class _Cuda(torch.Tensor):
    """A tensor that says it is on the current CUDA device."""

    def get_device(self):
        return 0


@pytest.mark.parametrize("change,error,text", [
    (dict(target_logits=torch.zeros(2, 4, 10, dtype=torch.float64)), TypeError, "fp32"), (dict(target_logits=torch.zeros(2, 10)), ValueError, "target_logits"),
    (dict(target_logits=torch.zeros(2, 0, 10)), ValueError, "target_logits"), (dict(draft_logits=torch.zeros(2, 4, 10)), ValueError, "draft_logits"),
    (dict(draft_logits=torch.zeros(2, 3, 10, dtype=torch.float16)), TypeError, "draft_logits"),
    (dict(tokens=torch.zeros(2, 3)), TypeError, "tokens"), (dict(tokens=torch.zeros(2, 4, dtype=torch.int64)), ValueError, "tokens"),
    (dict(uniforms=torch.zeros(2, 4, dtype=torch.float64)), TypeError, "uniforms"), (dict(uniforms=torch.zeros(2, 3)), ValueError, "uniforms"),
])
def test_verify_draft_checks_its_tensors(change, error, text, monkeypatch):
    from dropkv_b200 import paged
    monkeypatch.setattr(paged, "_current_device", lambda: 0)
    a = dict(target_logits=torch.zeros(2, 4, 10), tokens=torch.zeros(2, 3, dtype=torch.int64), uniforms=torch.zeros(2, 4)) | change
    with pytest.raises(error, match=text):
        verify_draft(**{k: v.as_subclass(_Cuda) for k, v in a.items()})


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        verify_draft(torch.zeros(2, 4, 10), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4))
