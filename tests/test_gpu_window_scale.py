"""The gradients of window attention do not depend on the scale of the values: what is kept of the output's rounding follows its size."""
import pytest
import torch

from test_gpu_window import inputs, plain, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-20, -60, 25])
def test_powers_of_two_change_nothing_in_bf16(power):
    """V times 2^p with dO times 2^-p: every product of the two, and with it dQ and dK, is the same number; O and dV carry the power."""
    q, k, v, g = inputs(torch.bfloat16, 2, 4, 2, 500, 500, 64, 31)
    want = run(q, k, v, g, 200, 3)
    got = run(q, k, v * 2.0 ** power, g * 2.0 ** -power, 200, 3)
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    assert torch.equal(got[0], want[0] * 2.0 ** power) and torch.equal(got[3], want[3] * 2.0 ** -power)


@pytest.mark.parametrize("dtype,power", [(torch.bfloat16, -20), (torch.bfloat16, 20), (torch.float16, -8), (torch.float16, 4)])
def test_error_of_the_gradients_at_other_scales(dtype, power):
    """dQ and dK are rounded twice, as dS and as themselves, by independent errors of the same relative size: sqrt(2) of one rounding's.
    Exponentials add squares below a tenth of that: 1.5 in all."""
    q, k, v, g = inputs(dtype, 2, 4, 4, 700, 700, 64, 15)
    v, g = v * 2.0 ** power, g * 2.0 ** -power
    want, _ = plain(q, k, v, g, 333, 3, 64 ** -0.5)
    got = run(q, k, v, g, 333, 3)
    for i in (1, 2):
        once = (want[i].to(dtype).double() - want[i]).norm()
        assert (got[i].double() - want[i]).norm() <= 1.5 * once, i
