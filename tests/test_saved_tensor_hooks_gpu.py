"""Hooks on the tensors that autograd keeps: what they bring back from the host serves as well as what was kept, and anything else is refused before a kernel
reads it."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

from simnets_tf_b200.ops.likelihood import log_probabilities
from simnets_tf_b200.ops.routing import route

pytestmark = pytest.mark.gpu


def answers(x):
    labels = torch.arange(x.shape[0] * x.shape[2], device="cuda").view(x.shape[0], x.shape[2]) % x.shape[1]
    got = log_probabilities(x, labels, 2, True)
    return [got.label, got.entropy, got.top]


CALLS = {"log probabilities": answers, "routing": lambda x: [route(x, top_k=2)[1]], "routing with sigmoids": lambda x: [route(x, top_k=2, sigmoid=True)[1]]}


def rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def logits(how):
    big = rand(3, 14, 10)
    return {"dense": lambda: big, "slice": lambda: big[:, 2:9, 1:8], "transposed": lambda: big.transpose(1, 2)}[how]().detach().requires_grad_()


@pytest.mark.parametrize("how", ["dense", "slice", "transposed"])
@pytest.mark.parametrize("name", sorted(CALLS))
def test_kept_on_the_host(name, how):
    """In the order in which the host keeps them, which is not that of a slice."""
    x = logits(how)
    plain = CALLS[name](x)
    gs = [rand(*y.shape, seed=1) for y in plain]
    want, = torch.autograd.grad(plain, x, gs)
    with save_on_cpu():
        kept = CALLS[name](x)
    have, = torch.autograd.grad(kept, x, gs)
    # (a value of the gradient is a handful of operations on what the forward pass left, whatever the order of the logits)
    assert torch.allclose(have, want, rtol=1e-6, atol=1e-6 * float(want.abs().max()))


def left_on_the_host(t):
    return t.cpu()


def shorter(t):
    return t.reshape(-1)[:-1]


def of_another_type(t):
    return t.double() if t.is_floating_point() else t.float()


@pytest.mark.parametrize("change", [left_on_the_host, shorter, of_another_type])
@pytest.mark.parametrize("name", sorted(CALLS))
def test_another_tensor_than_was_saved(name, change):
    x = logits("dense")
    kept, changed = [], None

    def pack(t):
        kept.append(t.detach())
        return len(kept) - 1

    def unpack(i):
        return change(kept[i]) if i == changed else kept[i]
    with saved_tensors_hooks(pack, unpack):
        outs = CALLS[name](x)
    gs = [torch.ones_like(y) for y in outs]
    want, = torch.autograd.grad(outs, x, gs, retain_graph=True)
    assert len(kept) >= 2
    for changed in range(len(kept)):
        with pytest.raises((RuntimeError, ValueError, TypeError), match="gave back|CPU kernels|same device|share a dtype|axis|labels|gradient"):
            torch.autograd.grad(outs, x, gs, retain_graph=True)
    changed = None
    assert bool((torch.autograd.grad(outs, x, gs)[0] == want).all())
