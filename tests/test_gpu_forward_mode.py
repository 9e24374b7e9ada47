"""Forward-mode differentiation: the rotation's tangent is the rotation of the tangent (the tolerance is that of the rotation
itself); an operator without one refuses dual tensors instead of dropping their tangent."""
import pytest
import torch
from torch.autograd import forward_ad

from lrqk_b200 import apply_rotary, rotary_frequencies
from test_gpu_rotary import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("adjoint", [False, True])
def test_tangents_of_the_rotation(dtype, interleaved, adjoint):
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    q, k, dq, dk = r(2, 4, 9, 64), r(2, 2, 9, 64), r(2, 9, 4, 64).transpose(1, 2), r(2, 2, 9, 64)
    inv, pos = rotary_frequencies(48, device="cuda")[0], torch.randint(-50, 5000, (2, 9), generator=g, device="cuda")
    kw = dict(factor=1.25, interleaved=interleaved, adjoint=adjoint)
    want = apply_rotary(q, k, pos, inv, **kw)
    with forward_ad.dual_level():
        for a, b in ((dq, dk), (dq, None), (None, dk)):
            x = q if a is None else forward_ad.make_dual(q, a)
            y = k if b is None else forward_ad.make_dual(k, b)
            got = [forward_ad.unpack_dual(z) for z in apply_rotary(x, y, pos, inv, **kw)]
            for z, w, d in zip(got, want, (a, b)):
                assert torch.equal(z.primal, w)
                if d is None:
                    assert z.tangent is None or not bool(z.tangent.any())
                else:
                    check(z.tangent, d, pos, inv, 1.25, interleaved, adjoint)
        with torch.no_grad():
            alone = forward_ad.unpack_dual(apply_rotary(forward_ad.make_dual(q, dq), None, pos, inv, **kw))
        check(alone.tangent, dq, pos, inv, 1.25, interleaved, adjoint)
        both = forward_ad.make_dual(q.clone().requires_grad_(), dq)     # a dual tensor that is also differentiated backwards
        out = forward_ad.unpack_dual(apply_rotary(both, None, pos, inv, **kw))
        check(out.tangent, dq, pos, inv, 1.25, interleaved, adjoint)
        assert out.primal.requires_grad


def test_function_transforms_are_refused_loudly():
    q, pos, inv = torch.ones(1, 1, 2, 8, device="cuda"), torch.arange(2, device="cuda"), rotary_frequencies(8, device="cuda")[0]
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: apply_rotary(x, None, pos, inv), (q,), (q,))


@pytest.mark.parametrize("which", range(5))
def test_tree_attention_refuses_dual_tensors(which):
    from lrqk_b200 import tree_attention
    x = [torch.randn(1, 2, n, 64, device="cuda") for n in (3, 8, 8, 3, 3)]
    want = tree_attention(*x)
    with forward_ad.dual_level():
        dual = list(x)
        dual[which] = forward_ad.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(ValueError, match="forward-mode"):
            tree_attention(*dual)
        assert torch.equal(tree_attention(*x), want)               # a level alone changes nothing
