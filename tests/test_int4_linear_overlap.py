"""int4_linear refuses an out over what its work-groups still read, on the host."""
import ctypes

import pytest
import torch

from pisceslx_amd import _lib

ROWS, K, O = 3, 300, 64
X, BIAS, CODES, SCALES, OUT = (0x100000 * i for i in range(1, 6))
CODE_BYTES, SCALE_BYTES = 4 * 3 * 1024, 4 * 3 * 32


def call(n=ROWS, x=X, bias=BIAS, codes=CODES, scales=SCALES, out=OUT):
    w = _lib.Int4Matrix(K, O, codes, scales)
    return _lib.lib().yvmoe_int4_linear(x, _lib.ACT_BF16, n, ctypes.byref(w), bias, out, None)


@pytest.mark.parametrize("over", [
    dict(out=BIAS), dict(out=BIAS + O * 2 - 2), dict(bias=OUT + (ROWS - 1) * O * 2), dict(n=1, out=BIAS + 2),
    dict(n=1, bias=OUT + 2), dict(out=CODES), dict(out=CODES + CODE_BYTES - 2), dict(codes=OUT + 128),
    dict(out=SCALES + SCALE_BYTES - 2), dict(scales=OUT + 8), dict(out=X), dict(out=X + ROWS * K * 2 - 2),
])
def test_refused(over):
    assert call(**over) == _lib.YVMOE_ERR_ARG, over
    assert b"overlaps" in _lib.lib().yvmoe_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the call would run on these addresses")
@pytest.mark.parametrize("beside", [
    dict(), dict(n=1, out=BIAS), dict(out=BIAS + O * 2), dict(bias=OUT + ROWS * O * 2), dict(out=CODES + CODE_BYTES),
    dict(out=SCALES + SCALE_BYTES), dict(out=X + ROWS * K * 2), dict(bias=None),
])
def test_neighbours_are_not_refused(beside):
    """Without a GPU the launch is what fails."""
    assert call(**beside) == _lib.YVMOE_ERR_LAUNCH


@pytest.mark.gpu
def test_one_row_onto_its_bias(cuda):
    from pisceslx_amd import functional as yvf
    from pisceslx_amd.quant import pack_linear
    from test_gpu_int4_linear import randn
    pk = pack_linear(randn(1, 200, 300, dtype=torch.float32))
    x, y = randn(2, 1, 300), randn(3, 1, 200)
    want = yvf.int4_linear(x, pk, y.clone())
    assert torch.equal(yvf.int4_linear(x, pk, y, out=y), want)
    rows = randn(4, 3, 200)
    with pytest.raises(ValueError, match="overlaps bias"):
        yvf.int4_linear(randn(5, 3, 300), pk, rows[1], out=rows)
