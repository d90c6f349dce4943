"""The feed-forward operators' argument checks without a GPU: what Python refuses before any device work, and what the C
ABI refuses before any CUDA call."""
import ctypes

import pytest
import torch

from _feedforward import decode, random_pair, table


def test_python_refuses_first():
    from mxq import nn
    g = torch.Generator().manual_seed(0)
    w = random_pair((6, 64), "MXFP8_E4M3", g, "cpu")
    x = random_pair((4, 64), "MXFP8_E4M3", g, "cpu")
    for text, call in (
            ("element format", lambda: nn.linear_packed(x, w, None)),
            ("scales of w", lambda: nn.linear_packed(x, (w[0], w[1][:5]), "MXFP8_E4M3")),
            ("activation", lambda: nn.linear_packed(x, w, "MXFP8_E4M3", activation="softplus")),
            ("bias must have", lambda: nn.linear_packed(x, w, "MXFP8_E4M3", bias=torch.zeros(3))),
            ("k must be", lambda: nn.route(torch.zeros(2, 4), 5)),
            ("n_experts", lambda: nn.dispatch(torch.zeros(2, 2, dtype=torch.int32), -1)),
            ("down", lambda: nn.MXExperts(torch.zeros(2, 8, 8), torch.zeros(3, 8, 4)))):
        with pytest.raises(ValueError, match=text):
            call()


def test_c_abi_refuses_first():
    from mxq import _lib
    L = _lib.lib()
    none = None

    def linear(M=4, N=4, K=64, x_pitch=64, w_pitch=64, x=64, **kw):
        s = dict(x_e=4, x_m=3, w_e=4, w_m=3, activation=0, out=0, out_e=0, out_m=0, x_type=0) | kw
        return L.mxq_linear_packed(x, none, x_pitch, M, 64, none, w_pitch, N, K, ctypes.byref(_lib.MxqProductSpec(**s)), none, none, 0,
                                   none, none, none, 0, none)
    for text, rc, call in (
            (b"no spec", _lib.ERR_VALUE, lambda: L.mxq_linear_packed(*[none] * 2, 0, 0, *[none] * 2, 0, 0, 0, none, *[none] * 2, 0,
                                                                     *[none] * 3, 0, none)),
            (b"bad sizes", _lib.ERR_VALUE, lambda: linear(K=0)),
            (b"bad sizes", _lib.ERR_VALUE, lambda: linear(M=-1)),
            (b"x has no MX element", _lib.ERR_VALUE, lambda: linear(x_e=3, x_m=3)),
            (b"type 5 of x", _lib.ERR_VALUE, lambda: linear(x_type=5)),
            (b"rows of w are 63 apart", _lib.ERR_VALUE, lambda: linear(w_pitch=63)),
            (b"pair up", _lib.ERR_VALUE, lambda: linear(w_e=2, w_m=1, K=63)),
            (b"a workspace of 384 bytes", _lib.ERR_VALUE, lambda: linear(x_pitch=74, w_pitch=80, K=72)),
            (b"a workspace of 256 bytes", _lib.ERR_VALUE, lambda: linear(x=8)),
            (b"a workspace of 256 bytes", _lib.ERR_VALUE, lambda: linear(w_e=2, w_m=3)),
            (b"a workspace of 384 bytes", _lib.ERR_VALUE, lambda: linear(x_type=2)),
            (b"activation", _lib.ERR_VALUE, lambda: linear(activation=9)),
            (b"output type", _lib.ERR_VALUE, lambda: linear(out=4)),
            (b"even number", _lib.ERR_VALUE, lambda: linear(N=5, activation=5)),
            (b"not an MX element", _lib.ERR_VALUE, lambda: linear(out=3, out_e=4, out_m=4)),
            (b"needs scales", _lib.ERR_VALUE, lambda: linear(out=3, out_e=4, out_m=3))):
        assert call() == rc and text in L.mxq_last_error(), (text, L.mxq_last_error())
    assert linear(M=0) == _lib.OK                             # nothing to do, no CUDA call
    spec = _lib.MxqProductSpec(4, 3, 4, 3, 0, 0, 0, 0, 0)

    def experts(E=2, slots=4, rows=2, per=2):
        return L.mxq_experts_packed(64, none, 64, rows, 64, none, 64, E, 4, 64, none, none, slots, per, ctypes.byref(spec), none, none,
                                    none, none, 0, none)
    fp4 = _lib.MxqProductSpec(2, 1, 2, 1, 0, 0, 0, 0, 0)
    assert L.mxq_product_workspace(64, 64, 10, 64, 64, 10, 128, 0, ctypes.byref(fp4)) == 0
    assert L.mxq_product_workspace(64, 64, 10, 64, 64, 10, 128, 20, ctypes.byref(fp4)) == 1280 + 2688   # widened and in order
    assert L.mxq_product_workspace(64, 64, 10, 64, 64, 10, 128, 1, none) == -1
    assert experts(E=1025) == _lib.ERR_UNSUPPORTED and b"1024 experts" in L.mxq_last_error()
    assert experts(rows=1) == _lib.ERR_VALUE and b"do not serve" in L.mxq_last_error()
    assert experts(slots=0) == _lib.OK

    def route(E=8, k=2, **kw):
        s = dict(score=0, groups=1, keep=1, top2=0, renormalize=0, scale=1.0) | kw
        return L.mxq_route(none, 0, 8, none, none, none, 0, E, k, ctypes.byref(_lib.MxqRouteSpec(**s)), none)
    assert route() == _lib.OK
    for text, kw in ((b"experts", dict(E=1025)), (b"k must be", dict(k=9)), (b"score", dict(score=2)), (b"groups", dict(groups=3)),
                     (b"groups", dict(groups=2, keep=3))):
        assert route(**kw) == _lib.ERR_VALUE and text in L.mxq_last_error()
    assert L.mxq_dispatch(none, -1, 4, none, none, none, none, 0, none) == _lib.ERR_VALUE
    assert L.mxq_dispatch(none, 4, 2000, none, none, none, none, 0, none) == _lib.ERR_VALUE
    assert L.mxq_dispatch_workspace(98304, 8) == 0 and L.mxq_dispatch_workspace(98305, 8) == 148 * 8 * 4
    assert L.mxq_dispatch(none, 98305, 8, none, none, none, none, 0, none) == _lib.ERR_VALUE and b"4736 bytes" in L.mxq_last_error()
    assert L.mxq_combine(none, 0, none, none, none, 0, none, 3, 0, 4, none) == _lib.ERR_VALUE
    assert L.mxq_combine(none, 7, none, none, none, 0, none, 3, 1, 4, none) == _lib.ERR_VALUE
    assert L.mxq_lay_codes(none, 8, 16, 24, 1, 8, 4, 3, none) == _lib.ERR_VALUE
    assert L.mxq_pack_rows(none, 9, 8, 16, 16, none, 1, 8, 4, 3, none) == _lib.ERR_VALUE


def test_tables_are_the_formats():
    """The tests' own decoder: the largest value and the count of special codes of each format."""
    for fmt, top, special in (("MXFP8_E4M3", 448.0, 2), ("MXFP8_E5M2", 57344.0, 8), ("MXFP6_E3M2", 28.0, 0), ("MXFP6_E2M3", 7.5, 0),
                              ("MXFP4", 6.0, 0)):
        t = table(fmt)
        assert float(t[t.isfinite()].max()) == top and int((~t.isfinite()).sum()) == special
    pair = (torch.tensor([[0x21, 0x7f]], dtype=torch.uint8), torch.tensor([[128]], dtype=torch.uint8))
    assert decode(pair, "MXFP4").tolist() == [[1.0, 2.0, -12.0, 12.0]]
