"""The stack's feed-forward block with its first half in one kernel, where that kernel cannot take part: forward derivatives, torch.func's
transforms, hooks, autocast and other modules in place of its projections."""

import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

from helpers import dev

pytestmark = pytest.mark.gpu


def blocks():
    from xlstm_hip.stack import _FFN
    torch.manual_seed(0)
    fused = _FFN(64, 96, fused=True).to(torch.bfloat16).to(dev())
    plain = _FFN(64, 96).to(torch.bfloat16).to(dev())
    plain.load_state_dict(fused.state_dict())
    x, t = (torch.randn(2, 9, 64, generator=torch.Generator().manual_seed(s)).to(torch.bfloat16).to(dev()) for s in (1, 2))
    return fused, plain, x, t


def test_forward_derivatives(gpu_case):
    fused, plain, x, t = blocks()
    found = []
    for ffn in (fused, plain):
        with forward_ad.dual_level():
            found.append(forward_ad.unpack_dual(ffn(forward_ad.make_dual(x, t))))
    assert torch.equal(found[0].primal, found[1].primal) and torch.equal(found[0].tangent, found[1].tangent)


def test_transforms(gpu_case):
    fused, plain, x, t = blocks()
    for transform in (lambda f: torch.func.jvp(f, (x,), (t,)), lambda f: (torch.func.grad(lambda y: f(y).float().sum())(x),),
                      lambda f: (torch.func.vmap(f)(x),)):
        for a, b in zip(transform(fused), transform(plain)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["forward", "forward_pre", "full_backward"])
@pytest.mark.parametrize("name", ["proj_up", "proj_up_gate"])
def test_hooks_run(gpu_case, kind, name):
    fused, _, x, _ = blocks()
    seen = []
    handle = getattr(getattr(fused, name), f"register_{kind}_hook")(lambda *a: seen.append(name))
    fused(x.requires_grad_(True)).float().sum().backward()
    assert seen == [name]
    handle.remove()


def test_other_modules_are_called(gpu_case):
    """A projection replaced by a module with a weight of its own kind (an adapter around it, say)."""
    class Twice(nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    fused, plain, x, _ = blocks()
    for ffn in (fused, plain):
        other = Twice(64, 96, bias=False).to(torch.bfloat16).to(dev())
        other.load_state_dict(ffn.proj_up.state_dict())
        ffn.proj_up = other
    with torch.no_grad():
        assert torch.equal(fused(x), plain(x))


def test_autocast(gpu_case):
    """Weights in float32 under autocast: the projections cast them."""
    fused, plain, x, _ = blocks()
    fused, plain = fused.float(), plain.float()
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(fused(x), plain(x))


def test_the_kernel_runs(gpu_case):
    """Without any of these it is the fused kernel's result, differentiated or not."""
    import xlstm_hip
    fused, _, x, _ = blocks()
    want = fused.proj_down(xlstm_hip.gated_linear_unit(x, fused.proj_up_gate.weight, fused.proj_up.weight))
    assert torch.equal(fused(x), want)
    with torch.no_grad():
        assert torch.equal(fused(x), want)
