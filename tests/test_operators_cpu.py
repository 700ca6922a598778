"""Host-side argument handling of the attention and multi-axis rotary entry
points. CPU only: no kernel is launched here."""
import ctypes

import pytest
import torch

import bloth_b200
from bloth_b200 import _lib


def test_axes_in_sections():
    assert bloth_b200.mrope_axes([2, 1, 1]) == (0, 0, 1, 2)
    assert bloth_b200.mrope_axes([16, 24, 24]) == (0,) * 16 + (1,) * 24 + (2,) * 24
    assert bloth_b200.mrope_axes([3]) == (0, 0, 0)


def test_axes_interleaved():
    # Qwen3-VL: h at 1, 4, 7, ..., w at 2, 5, 8, ..., time everywhere else
    axes = bloth_b200.mrope_axes([24, 20, 20], interleaved=True)
    assert axes[:6] == (0, 1, 2, 0, 1, 2) and axes[60:] == (0, 0, 0, 0)
    assert [axes.count(a) for a in range(3)] == [24, 20, 20]
    with pytest.raises(ValueError):
        bloth_b200.mrope_axes([2, 10, 10], interleaved=True)


@pytest.mark.parametrize("bad", [[], [1, 1, 1, 1, 1], [4, -1]])
def test_axes_refused(bad):
    with pytest.raises(ValueError):
        bloth_b200.mrope_axes(bad)


def test_cpu_tensors_are_refused():
    q, k = torch.randn(1, 4, 2, 64), torch.randn(1, 4, 1, 64)
    with pytest.raises(AssertionError, match="CUDA GPU required"):
        bloth_b200.fused_attention(q, k, k)
    with pytest.raises(AssertionError, match="CUDA GPU required"):
        bloth_b200.apply_mrope_qk(q, k, torch.zeros(3, 1, 4).long(), torch.ones(32), (0,) * 32)


def _fwd(**kw):
    """bloth_attention_fwd with NULL tensors and one argument changed."""
    a = dict(q_seq=None, k_seq=None, seq_dtype=_lib.I32, packed=0, B=1, Sq=4, Sk=4, Hq=2, Hk=1,
             D=64, scale=0.125, causal=1, window=0, dtype=_lib.BF16)
    a.update(kw)
    return _lib.load().bloth_attention_fwd(
        None, None, None, None, None, None, None, None, None, None, a["q_seq"], a["k_seq"],
        a["seq_dtype"], a["packed"], a["B"], a["Sq"], a["Sk"], a["Hq"], a["Hk"], a["D"],
        a["scale"], a["causal"], a["window"], a["dtype"], None, 0, None)


def test_attention_status_codes():
    dummy = _lib.ptr(torch.zeros(4, dtype=torch.int32))
    assert _fwd() == 5  # NULL tensors
    assert _fwd(Sq=0) == 0 and _fwd(B=0) == 0  # nothing to do
    assert _fwd(dtype=_lib.I32) == 1
    for bad in (dict(D=96), dict(Hq=3, Hk=2), dict(Hk=0), dict(B=-1), dict(Sq=-1), dict(Sk=2 ** 40),
                dict(packed=2, B=2), dict(packed=-1)):
        assert _fwd(**bad) == 2, bad
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(window=-1), dict(window=3, causal=0)):
        assert _fwd(**bad) == 7, bad
    assert _fwd(packed=1) == 5
    assert _fwd(k_seq=dummy, seq_dtype=_lib.F32) == 1


def test_attention_workspace_sizes():
    lib = _lib.load()
    f = lib.bloth_attention_bwd_workspace_bytes
    # two fp32 statistics for every query row, in tiles of 128
    assert f(2, 200, 300, 4, 2, 64, 0, _lib.BF16) >= 2 * 4 * 2 * 200 * 4
    assert f(1, 200, 300, 4, 2, 64, 5, _lib.BF16) >= 2 * 4 * 200 * 4
    assert f(1, 200, 300, 4, 3, 64, 0, _lib.BF16) == 0  # refused sizes need nothing
    assert f(1, 0, 300, 4, 2, 64, 0, _lib.BF16) == 0


def test_mrope_status_codes():
    lib = _lib.load()
    st = _lib.strides((0, 0, 0))
    one = _lib.ptr(torch.zeros(4))
    axes = (ctypes.c_uint8 * 32)()

    def call(pos=one, pos_st=st, n=3, of=axes, inv=one, D=64):
        return lib.bloth_mrope(None, st, None, st, None, None, None, None, pos, pos_st, _lib.I64,
                               n, of, inv, 1.0, 1, 1, 1, 0, D, 0, _lib.BF16, None)

    assert call() == 5  # NULL tensors
    assert call(n=0) == 2 and call(n=5) == 2 and call(D=96) == 2
    assert call(pos=None) == 5 and call(pos_st=None) == 5 and call(of=None) == 5
    assert call(inv=None) == 5
    bad = (ctypes.c_uint8 * 32)(*([3] * 32))
    assert call(of=bad) == 7
