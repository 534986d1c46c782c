"""What the paged operators refuse, without a GPU: the C entries' argument checks
(placeholder pointers that are never followed) and the Python checks."""

import pytest
import torch

from dropkv_b200 import (_lib, block_tables, qk_norm_rope, store_rows, token_logprobs, tree_attention,
                         tree_mask_from_parents)

P = 4096  # a placeholder device address


def _refused(rc, code, text):
    assert rc == code and text in _lib.load().dropkv_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(lens=None), "NULL"), (dict(table=None), "NULL"), (dict(slots=None), "slots"), (dict(free=None), "free_blocks"),
    (dict(B=0), "B must be"), (dict(B=65536), "B must be"), (dict(block=0), "block_size"), (dict(max_blocks=0), "max_blocks"),
    (dict(max_new=-1), "max_new"), (dict(n_free=-1), "n_free"), (dict(held=P), "go together"),
    (dict(table_in=P), "go together"), (dict(table_in=P, held=P, stride=3), "shorter"),
])
def test_block_tables_refuses(change, text):
    a = dict(lens=P, new=None, table_in=None, stride=4, held=None, B=2, block=16, free=P, n_free=5, max_blocks=4,
             max_new=8, table=P, held_out=P, slots=P, used=P) | change
    rc = _lib.load().dropkv_block_tables(*a.values(), None)
    _refused(rc, _lib.ERR_ARG, text)


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "NULL"), (dict(slots=None), "NULL"), (dict(vp=None), "NULL"), (dict(eb=3), "elem_bytes"),
    (dict(B=-1), "sizes"), (dict(D=0), "sizes"), (dict(block=0), "sizes"), (dict(k=P + 1), "aligned"),
])
def test_store_rows_refuses(change, text):
    a = dict(k=P, v=P, slots=P, kp=P, vp=P, pages=4, block=16, eb=2, B=1, H=2, N=3, D=64) | change
    s = (1, 1, 1)
    rc = _lib.load().dropkv_store_rows(a["k"], *s, a["v"], *s, a["slots"], a["kp"], *s, a["vp"], *s, a["pages"],
                                       a["block"], a["eb"], a["B"], a["H"], a["N"], a["D"], None)
    _refused(rc, _lib.ERR_ARG, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=7), _lib.ERR_ARG, "dtype"), (dict(q=None), _lib.ERR_ARG, "NULL"), (dict(pos=None), _lib.ERR_ARG, "NULL"),
    (dict(R=3), _lib.ERR_ARG, "even"), (dict(R=130), _lib.ERR_ARG, "even"), (dict(cos=None), _lib.ERR_ARG, "cos"),
    (dict(eps=-1.0), _lib.ERR_ARG, "eps"), (dict(eps=float("nan")), _lib.ERR_ARG, "eps"),
    (dict(D=1025), _lib.ERR_UNSUPPORTED, "1024"), (dict(Hq=0), _lib.ERR_ARG, "sizes"),
    (dict(slots=P), _lib.ERR_ARG, "slots need"), (dict(q=P + 1), _lib.ERR_ARG, "aligned"),
])
def test_qk_norm_rope_refuses(change, code, text):
    a = dict(q=P, k=P, eps=1e-6, cos=P, R=128, pos=P, dtype=2, Hq=8, D=128, slots=None) | change
    s = (1, 1, 1)
    rc = _lib.load().dropkv_qk_norm_rope(a["q"], *s, a["k"], *s, None, None, a["eps"], a["cos"], P, 10, a["R"], 0,
                                         a["pos"], 0, a["dtype"], 1, a["Hq"], 2, 3, a["D"], P, P, None, *s, a["slots"],
                                         None, *s, None, *s, 0, 1, None)
    _refused(rc, code, text)


@pytest.mark.parametrize("change,code,text", [
    (dict(q=None), _lib.ERR_ARG, "NULL"), (dict(k=None), _lib.ERR_ARG, "K and V"), (dict(out=None), _lib.ERR_ARG, "NULL"),
    (dict(dtype=0), _lib.ERR_UNSUPPORTED, "bf16 or fp16"), (dict(D=96), _lib.ERR_UNSUPPORTED, "64 or 128"),
    (dict(T=257), _lib.ERR_UNSUPPORTED, "256 nodes"), (dict(T=0), _lib.ERR_ARG, "sizes"), (dict(Hq=6), _lib.ERR_ARG, "sizes"),
    (dict(B=20000), _lib.ERR_ARG, "sizes"), (dict(k=P + 8), _lib.ERR_ARG, "16-byte"), (dict(k_ss=100), _lib.ERR_ARG, "16-byte"),
    (dict(k_ss=64), _lib.ERR_ARG, "strides"), (dict(scale=0.0), _lib.ERR_ARG, "scale"),
    (dict(scale=float("nan")), _lib.ERR_ARG, "scale"), (dict(table=P, block=24), _lib.ERR_UNSUPPORTED, "power of two"),
    (dict(table=P, block=4), _lib.ERR_UNSUPPORTED, "power of two"), (dict(table=P, block=2048), _lib.ERR_UNSUPPORTED, "power of two"),
    (dict(table=P, block=16), _lib.ERR_ARG, "max_blocks"), (dict(), _lib.ERR_WORKSPACE, "workspace"),
])
def test_tree_attention_refuses(change, code, text):
    a = dict(q=P, k=P, k_ss=128, table=None, max_blocks=3, block=0, dtype=2, B=1, Hq=32, T=5, D=128, cap=4000, scale=0.1,
             out=P) | change
    lib = _lib.load()
    if change == {} and lib.dropkv_tree_attention_workspace_size(1, 32, 8, 5, 128, 4000) == 0:
        pytest.skip("no workspace needed")
    rc = lib.dropkv_tree_attention(a["q"], 1, 1, 1, 1, a["k"], 4000 * 1024, 4000 * 128, a["k_ss"], P, 4000 * 1024,
                                   4000 * 128, 128, a["table"], a["max_blocks"], a["block"], 9, P, None, 0, 0, 0,
                                   a["dtype"], a["B"], a["Hq"], 8, a["T"], a["D"], a["cap"], a["scale"], a["out"], None,
                                   0, None)
    _refused(rc, code, text)


@pytest.mark.parametrize("scale", [float("inf"), 3e38])
def test_tree_attention_refuses_scales_that_are_no_number(scale):
    # infinity times a score of 0, or less another infinity, is NaN: no output could be told from a fault
    lib = _lib.load()
    need = lib.dropkv_tree_attention_workspace_size(1, 1, 1, 1, 64, 8)
    s = (512, 512, 64)
    rc = lib.dropkv_tree_attention(P, 64, 64, 64, 1, P, *s, P, *s, None, 0, 0, 0, P, None, 0, 0, 0, 2, 1, 1, 1, 1, 64, 8,
                                   scale, P, P, need, None)
    _refused(rc, _lib.ERR_ARG, "scale")


@pytest.mark.parametrize("B,max_blocks,block,text", [
    (1, (1 << 28) - 1, 8, "too long"), (1, (1 << 25) - 1, 64, "too long"),   # capacities a tile short of 2^31
    (128, (1 << 21) - 64, 1024, "too many tiles"),                          # the last CTA's share would end past 2^31
    (512, 1 << 20, 1024, "too many tiles"),
])
def test_tree_attention_refuses_lines_of_tiles_past_31_bits(B, max_blocks, block, text):
    lib, cap = _lib.load(), max_blocks * block
    need = lib.dropkv_tree_attention_workspace_size(B, 1, 1, 1, 64, cap)
    s = (1 << 20, 1 << 20, 64)
    rc = lib.dropkv_tree_attention(P, 64, 64, 64, 1, P, *s, P, *s, P, max_blocks, block, 9, P, None, 0, 0, 0, 2, B, 1, 1, 1,
                                   64, cap, 0.1, P, P, need, None)
    _refused(rc, _lib.ERR_UNSUPPORTED, text)


@pytest.mark.parametrize("change,text", [
    (dict(logits=None), "NULL"), (dict(tokens=None), "NULL"), (dict(dtype=5), "dtype"), (dict(V=0), "sizes"),
    (dict(top=65), "top_k"), (dict(top=-1), "top_k"), (dict(top=11, V=10), "top_k"), (dict(tau=0.0), "temperature"),
    (dict(tau=float("inf")), "temperature"), (dict(tau=float("nan")), "temperature"), (dict(stride=-5), "row_stride"),
    (dict(logits=P + 1), "aligned"),
])
def test_token_logprobs_refuses(change, text):
    a = dict(logits=P, stride=1000, dtype=2, N=3, V=1000, tokens=P, top=5, tau=1.0) | change
    rc = _lib.load().dropkv_token_logprobs(a["logits"], a["stride"], a["dtype"], a["N"], a["V"], a["tokens"], 1, a["top"],
                                           a["tau"], P, P, P, P, None, 0, None)
    _refused(rc, _lib.ERR_ARG, text)


def test_workspaces_of_invalid_problems_are_empty():
    lib = _lib.load()
    assert lib.dropkv_tree_attention_workspace_size(1, 6, 4, 5, 128, 100) == 0
    assert lib.dropkv_tree_attention_workspace_size(1, 8, 4, 300, 128, 100) == 0
    assert lib.dropkv_token_logprobs_workspace_size(4, 100, 101) == 0


def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(1, 2, 3, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        block_tables(i, 16, i, 4, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        store_rows(x, x, torch.zeros(1, 3, dtype=torch.int64), x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        qk_norm_rope(x, x, x[0, 0], x[0, 0], torch.arange(3))
    with pytest.raises(RuntimeError, match="CUDA"):
        tree_attention(x, x, x, i[:1])
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(x[0, 0], torch.arange(3))


class _OnDevice(torch.Tensor):
    """A tensor that says it is on CUDA device 3."""

    def get_device(self):
        return 3


@pytest.mark.parametrize("op,arguments", [
    (block_tables, dict(block_size=16, max_blocks=4, lens=None, free_blocks=None, max_new=4)),
    (store_rows, dict(slots=None, K=None, V=None, K_pages=None, V_pages=None)),
    (qk_norm_rope, dict(eps=1e-5, interleaved=True, q_weight="none", Q=None, K=None, cos=None, sin=None, positions=None)),
    (tree_attention, dict(scale=0.1, tree_mask="none", Q=None, K=None, V=None, cache_lens=None)),
    (token_logprobs, dict(top_k=5, temperature=0.5, logits=None, tokens=None)),
])
def test_calls_enter_their_tensors_device_however_the_arguments_are_given(op, arguments, monkeypatch):
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
    monkeypatch.setattr(paged, "_current_device", lambda: 3)   # the current one is not entered again
    with pytest.raises((ValueError, TypeError, RuntimeError, IndexError)):
        op(**arguments)
    assert entered == [3]


def test_tree_masks_from_parents():
    par = torch.tensor([[-1, 0, 0, 1, -1, 4], [-1, 0, 1, 2, 3, 4]])
    mask, depth = tree_mask_from_parents(par)
    for b in range(2):
        for i in range(6):
            want, j = {i}, int(par[b, i])
            while j >= 0:
                want.add(j)
                j = int(par[b, j])
            assert set(mask[b, i].nonzero()[:, 0].tolist()) == want and int(depth[b, i]) == len(want) - 1
    one, d = tree_mask_from_parents(torch.tensor([-1]))
    assert one.tolist() == [[True]] and d.tolist() == [0]
