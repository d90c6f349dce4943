"""The products through the C ABI, as callers with memory of their own make them: rows of x further apart than their codes, a
workspace of exactly the bytes asked for with a guard behind it, x that ends with its last code."""
import ctypes

import pytest
import torch

from _feedforward import random_pair

pytestmark = pytest.mark.gpu
DEV = "cuda"


def pitched(codes, pitch):
    """codes (rows x K) with their rows `pitch` bytes apart, 0x7f (NaN in E4M3) between them, the last one ending the buffer."""
    rows, K = codes.shape
    flat = torch.full(((rows - 1) * pitch + K,), 0x7f, dtype=torch.uint8, device=DEV)
    flat.as_strided((rows, K), (pitch, 1)).copy_(codes)
    return flat


@pytest.mark.parametrize("K,pitch", [(128, 4096), (64, 80), (40, 48), (1000, 1008), (1000, 2048), (2048, 2048)])
@pytest.mark.parametrize("T,k,E", [(700, 3, 4), (40, 2, 2), (9, 2, 5)])     # sorted first by tiles of 256 and of 64 rows; fetched one by one
def test_pitched_rows_through_a_plan(K, pitch, T, k, E):
    """The same bits as with x contiguous; nothing behind the workspace is written."""
    from mxq import _lib, nn
    g = torch.Generator().manual_seed(K + T)
    N, guard = 96, 1 << 20
    x, w = random_pair((T, K), "MXFP8_E4M3", g, DEV), random_pair((E, N, K), "MXFP8_E4M3", g, DEV)
    plan = nn.dispatch(torch.randint(-1, E, (T, k), generator=g).int().to(DEV), E)
    want = nn.experts_packed(x, w, "MXFP8_E4M3", plan, out=torch.float32)
    live = int(plan.offsets[-1])

    far, lib = pitched(x[0], pitch), _lib.lib()
    spec = _lib.MxqProductSpec(4, 3, 4, 3, 0, 0, 0, 0, 0)
    need = lib.mxq_product_workspace(_lib.ptr(far), pitch, T, _lib.ptr(w[0]), K, E * N, K, T * k, ctypes.byref(spec))
    space = torch.full((need + guard,), 0xa5, dtype=torch.uint8, device=DEV)
    y = torch.empty(T * k, N, device=DEV)
    _lib.call("mxq_experts_packed", _lib.ptr(far), _lib.ptr(x[1]), pitch, T, _lib.ptr(w[0]), _lib.ptr(w[1]), K, E, N, K,
              _lib.ptr(plan.offsets), _lib.ptr(plan.order), T * k, k, ctypes.byref(spec), None, _lib.ptr(y), None, _lib.ptr(space), need,
              _lib.stream(y.device))
    assert (space[need:] == 0xa5).all()
    assert torch.equal(y[:live], want[:live])


@pytest.mark.parametrize("residual", [False, True])
def test_rows_of_more_than_2_31_bytes(residual):
    """Float32 rows of y whose bytes pass 32 bits: every column is where it belongs, the residual's too."""
    from mxq import nn
    M, N, K = 2, (1 << 29) + 320, 32
    x = (torch.full((M, K), 0x38, dtype=torch.uint8, device=DEV), torch.full((M, 1), 127, dtype=torch.uint8, device=DEV))    # ones
    w = (torch.zeros(N, K, dtype=torch.uint8, device=DEV), torch.full((N, 1), 127, dtype=torch.uint8, device=DEV))
    at = torch.tensor([0, 77, 1 << 28, (1 << 29) - 1, 1 << 29, (1 << 29) + 33, N - 1], device=DEV)
    w[0][at] = 0x38
    r = torch.zeros(M, N, device=DEV) if residual else None
    if residual:
        r[1, at] = torch.arange(1, 8, dtype=torch.float32, device=DEV)
        r[0, N - 65] = 5.0
    y = nn.linear_packed(x, w, "MXFP8_E4M3", residual=r, out=torch.float32)
    assert (y[0, at] == K).all()
    assert torch.equal(y[1, at], K + torch.arange(1, 8, device=DEV) * float(residual))
    assert int(y.count_nonzero()) == 14 + int(residual)
    if residual:
        assert y[0, N - 65] == 5.0
