"""The packed products' waits run out instead of hanging: the test-only entry point makes every stage expect bytes that never
come, under a short limit. Every role leaves, y is NaN, the wait-status word and the device counter rise, the next call raises
until the word is cleared, and then the products are right again (no TMEM and no barrier is left behind)."""
import ctypes

import pytest
import torch

from _feedforward import assert_close, decode, product64, random_pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(4, 700, 1024), (700, 3000, 640)])       # few rows over clusters; pairs of CTAs, many tiles
def test_waits_run_out(M, N, K):
    from mxq import _lib, nn
    g = torch.Generator().manual_seed(M)
    x, w = random_pair((M, K), "MXFP8_E4M3", g, "cuda"), random_pair((N, K), "MXFP8_E4M3", g, "cuda")
    word, count = _lib.wait_word(), ctypes.c_uint32(0)
    assert word.value == 0
    _lib.call("mxq_device_timeouts", ctypes.byref(count))
    before = count.value
    y = torch.zeros(M, N, device="cuda")
    _lib.call("mxq_testing_product_timeout", _lib.ptr(x[0]), _lib.ptr(x[1]), M, _lib.ptr(w[0]), _lib.ptr(w[1]), N, K, _lib.ptr(y), 1 << 20,
              _lib.stream(y.device))
    torch.cuda.synchronize()
    try:
        assert word.value >= 1
        _lib.call("mxq_device_timeouts", ctypes.byref(count))
        assert count.value - before == word.value
        assert y.isnan().all()
        with pytest.raises(RuntimeError, match="gave up"):
            nn.linear_packed(x, w, "MXFP8_E4M3")
    finally:
        torch.cuda.synchronize()
        _lib.clear_waits()
    for _ in range(3):
        y = nn.linear_packed(x, w, "MXFP8_E4M3", out=torch.float32)
        assert_close(y, *product64(decode(x, "MXFP8_E4M3"), decode(w, "MXFP8_E4M3")), torch.float32)
    assert word.value == 0
