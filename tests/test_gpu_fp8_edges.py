"""``ccq_fp8_linear`` and the norms into 8 bits at the edges of each way that they run: strides of outputs, scales far from one,
numbers that are not finite, more wide rows than workgroups.  Which way a size takes is asserted, as in
``test_gpu_fp8_paths.py``, whose whole numbers these are: outputs have to be equal bit for bit."""

import ctypes

import pytest
import torch

from test_gpu_fp8_paths import ACTS, BF, DTYPES, FL, HF, _cuda, plan, whole

pytestmark = pytest.mark.gpu


def _bytes(t):
    return t.contiguous().view(torch.uint8)


#        M, N, K            act, dtype, way
ROWS = [((5, 300, 1030), None, BF, "0/8"), ((5, 300, 1030), "swiglu", HF, "0/8"), ((33, 4100, 2000), "relu", FL, "0/2"),
        ((900, 300, 600), None, BF, "64"), ((600, 1100, 700), "relu", FL, "64"), ((1100, 520, 90), "swiglu", HF, "64"),
        ((8192, 4096, 300), None, BF, "128"), ((3001, 2101, 250), "swiglu", BF, "128"), ((4500, 8300, 128), "relu", HF, "128"),
        ((16300, 2040, 2100), None, BF, "256"), ((16301, 2047, 4100), "relu", BF, "256"),
        ((16300, 2040, 2100), "swiglu", HF, "256")]


@pytest.mark.parametrize("size,act,dtype,way", ROWS, ids=str)
def test_output_rows_apart(size, act, dtype, way):
    """Rows of y at a stride of their own are those of a contiguous y, and nothing is written between them."""
    from ccq_amd import _lib
    M, N, K = size
    print("test_output_rows_apart", size, act, dtype, flush=True)
    assert plan(M, N, K, act, dtype, 0) == way
    dev, lib = _cuda(), _lib.load()
    gen = torch.Generator().manual_seed(M + N + K)
    x, w = whole(gen, M, K, dev), whole(gen, 2 * N if act == "swiglu" else N, K, dev)
    res = torch.randint(-9, 10, (M, N), generator=gen).to(dtype).to(dev)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def call(y, ldy):
        args = [v for t in (*x, *w) for v in (t.data_ptr(), t.stride(0))]
        assert lib.ccq_fp8_linear(*args, None, 0, res.data_ptr(), N, y.data_ptr(), ldy, None, 0, None, M, N, K, ACTS[act],
                                  DTYPES[dtype], st) == 0

    want = torch.empty(M, N, dtype=dtype, device=dev)
    call(want, N)
    for ldy in (0, N + 1, N + 24):
        big = torch.full((M * max(ldy, N) + 64,), -77.0, dtype=dtype, device=dev)
        call(big, ldy)
        torch.cuda.synchronize()
        rows = big[:M * max(ldy, N)].view(M, -1)
        assert torch.equal(_bytes(rows[:, :N]), _bytes(want)), ldy
        assert bool((rows[:, N:] == -77).all()) and bool((big[M * max(ldy, N):] == -77).all()), ldy
