"""What the recurrent agent's operators refuse, and how: types, shapes and devices are checked on the host, before any allocation or
launch (no GPU needed)."""
import pytest
import torch

from ac_solver.agents import recurrence as R


def scan_args(T=3, N=2, D=4, dtype=torch.float32):
    return torch.zeros(T, N, D, dtype=dtype), torch.zeros(T, N, D, dtype=dtype)


def test_the_scan_refuses_what_it_cannot_read():
    c, z = scan_args()
    ok = dict(reset=torch.zeros(3, 2, dtype=torch.bool), state=torch.zeros(2, 4))
    with pytest.raises(ValueError, match="GPU"):  # everything in order but the place
        R.gated_scan(c, z, **ok)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        R.gated_scan(c.double(), z.double())
    with pytest.raises(TypeError, match="tensor"):
        R.gated_scan([1.0], z)
    with pytest.raises(ValueError, match="gate is"):
        R.gated_scan(c, z.half())
    with pytest.raises(ValueError, match="gate has the shape"):
        R.gated_scan(c, z[:2])
    with pytest.raises(ValueError, match="steps, rows, features"):
        R.gated_scan(c[0], z[0])
    with pytest.raises(ValueError, match="at least one step"):
        R.gated_scan(c[:0], z[:0])
    with pytest.raises(ValueError, match="reset has the shape"):
        R.gated_scan(c, z, reset=ok["reset"].t())
    with pytest.raises(TypeError, match="reset"):
        R.gated_scan(c, z, reset=torch.zeros(3, 2))
    with pytest.raises(TypeError, match="state"):
        R.gated_scan(c, z, state=torch.zeros(2, 4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="state has the shape"):
        R.gated_scan(c, z, state=torch.zeros(1, 4))


def test_the_scan_gradient_refuses_what_does_not_fit_its_forward_pass():
    c, z = scan_args()
    with pytest.raises(ValueError, match="GPU"):
        R.gated_scan_backward(c, None, c, z, None, torch.zeros(8))


def test_scan_buffer_sizes():
    from ac_solver import _acx

    assert _acx.lib.acx_scan_bounds_bytes(1, 2, 4) == 32 and _acx.lib.acx_scan_bounds_bytes(17, 2, 4) == 64 and _acx.lib.acx_scan_bounds_bytes(16, 0, 4) == 0
    assert _acx.lib.acx_scan_workspace_bytes(1, 1, 1, _acx.F32) == 0 and _acx.lib.acx_scan_workspace_bytes(1 << 16, 1, 256, _acx.BF16) > 0
    assert _acx.lib.acx_scan_workspace_bytes(32, 131072, 256, _acx.F32) == 0
