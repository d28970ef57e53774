"""What gdn2_short_conv_step(inplace=True) gives back."""
import pytest
import torch

from test_short_conv_gpu import BF16, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,held", [(F32, F32), (BF16, BF16), (torch.float16, F32),
                                        (torch.float64, F32)])
def test_in_place_is_the_state(dev, dtype, held):
    """The state itself, also where x is of a type that is widened and the state of the one that is
    computed in; so that a loop which passes on what it gets goes on in place."""
    import gdn2_package as gp
    x = torch.randn((6, 3, 24), device=dev).to(dtype)
    w = torch.randn((24, 4), device=dev)
    state = torch.zeros((3, 3, 24), dtype=held, device=dev)
    whole, last = gp.gdn2_short_conv(x.transpose(0, 1), w)
    s = state
    for i in range(6):
        y, s = gp.gdn2_short_conv_step(x[i], w, state=s, inplace=True)
        assert s is state and y.dtype == dtype and torch.equal(y, whole[:, i])
    assert torch.equal(state.to(dtype), last)
    y, new = gp.gdn2_short_conv_step(x[0], w, state=state)
    assert new is not state and new.dtype == dtype
