"""The MEX gradients read the layer's output: one of another size is refused."""
import pytest
import torch

from simnets_tf_b200.ops.mex import mex, mex_backward, mex_forward, mex_input_grad, mex_offsets_grad

pytestmark = pytest.mark.gpu
KW = dict(blocks=[2, 1, 1], strides=[2, 1, 1], epsilon=0.5, use_unshared_regions=False)


@pytest.mark.parametrize("call", [mex_input_grad, mex_offsets_grad, mex_backward])
def test_an_output_of_another_size(call):
    x, off = torch.randn(2, 4, 6, 6, device="cuda"), torch.randn(1, 3, 2, 1, 1, device="cuda")
    y = mex_forward(x, off, 3, **KW)
    dy = torch.randn_like(y)
    for bad in (y[:1], y[:, :, ::2], y[..., :5], torch.zeros(0, device="cuda")):
        with pytest.raises(ValueError, match="orig_output must have shape"):
            call(x, off, bad, dy, 3, **KW)
    # the pooled gradient takes the output as it was before the pooling
    small = torch.randn(2, y.shape[1], 3, 3, device="cuda")
    with pytest.raises(ValueError, match="orig_output must have shape"):
        call(x, off, small, small, 3, pooled=True, **KW)
    call(x, off, y, small, 3, pooled=True, **KW)
    call(x, off, y.reshape(-1), dy, 3, **KW)


def test_an_output_that_a_hook_cut():
    x, off = torch.randn(2, 4, 6, 6, device="cuda", requires_grad=True), torch.randn(1, 3, 2, 1, 1, device="cuda")
    values = 2 * 6 * 6 * 6
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), lambda t: t.reshape(-1)[:-1] if t.numel() == values else t):
        y = mex(x, off, 3, **KW)
    assert y.numel() == values != x.numel()
    with pytest.raises(RuntimeError, match="orig_output must have shape"):       # (the engine's own kind, whatever a node throws)
        y.sum().backward()
