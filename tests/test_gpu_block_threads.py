"""The C ABI of the row kernels from several host threads, which hold no interpreter lock in the call."""

import struct
import threading

import pytest
import torch

from recap_b200 import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _norm_rows(x, y, out, h):
    """Packed recap_norm_rows_args: residual sum of fp32 rows [1, 1, C] and the root mean square norm of the sum."""
    c = x.shape[-1]
    return struct.Struct("<4Q8q3Q6q4Q10i2f").pack(
        x.data_ptr(), y.data_ptr(), out.data_ptr(), h.data_ptr(), *[c, c] * 4, 0, 0, 0, *[0] * 6, 0, 0, 0, 0, 1, 1, c, 2, 2, 1,
        0, 0, 0, 0, 1e-6, 1e-6)


def _rotate(x, out):
    """Packed recap_rotate_qk_args: norm over the heads of one token [1, heads, 1, 128], fp32."""
    heads = x.shape[1]
    strides = [heads * 128, 128, heads * 128]
    return struct.Struct("<4Q12qQ3qq4Q10i2f").pack(
        x.data_ptr(), 0, out.data_ptr(), 0, *strides, *[0] * 3, *strides, *[0] * 3, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, heads, 0, 1,
        128, 2, 2, 3, 0, 0, 1e-6, 1e-6)


@pytest.mark.parametrize("what", ["norm", "rotate"])
def test_calls_of_different_sizes_from_two_threads(what):
    """Rows of 8200 and of 16376 values, 128 heads and 100: the same kernel with more or less shared memory a block."""
    lib = _lib.load()
    if what == "norm":
        data = [[torch.randn(1, 1, c, device=DEV) for _ in range(4)] for c in (8200, 16376)]
        calls = [lambda s, a=_norm_rows(*t): lib.recap_norm_rows(a, s) for t in data]
    else:
        data = [[torch.randn(1, h, 1, 128, device=DEV) for _ in range(2)] for h in (100, 128)]
        calls = [lambda s, a=_rotate(*t): lib.recap_rotate_qk(a, None, s) for t in data]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    bad = [0, 0]

    def work(i):
        for n in range(20000):
            bad[i] += calls[i](streams[i].cuda_stream) != _lib.RECAP_OK
            if n % 500 == 499:
                streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert bad == [0, 0]
    for t in data:
        x = t[0].double() + (t[1].double() if what == "norm" else 0)
        dims = (-1,) if what == "norm" else (1, 3)
        want = x / torch.sqrt((x * x).mean(dims, keepdim=True) + 1e-6)
        # sums of up to 2^14 values over threads, lanes and warps (53 additions), the products, the result's rounding: 2^-24 each
        assert bool(((t[-1].double() - want).abs() <= 80 * 2.0**-24 * want.abs()).all())
