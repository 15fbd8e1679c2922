"""What the training operators promise about autograd, sizes and layouts, beside their values: derivatives that they do not
have are refused, limits are told by the forward call, any strides are taken."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from _training import inputs

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def test_forward_mode_is_refused():
    from sageattention import rotary_axes, sageattn_backward, sageattn_train

    q, k, v, dout = inputs(1, 2, 2, 40, 40, 64, BF16, "HND")
    pos = torch.arange(40, device="cuda")[:, None]
    out, lse = sageattn_train(q, k, v, return_lse=True)
    leaf = q.clone().requires_grad_(True)
    with fwad.dual_level():
        dq, dk, dd = (fwad.make_dual(x, torch.ones_like(x)) for x in (q, k, dout))
        calls = [("sageattn_train", lambda: sageattn_train(dq, k, v)), ("sageattn_train", lambda: sageattn_train(q, k, dk)),
                 ("sageattn_train", lambda: sageattn_train(leaf, dk, v)), ("rotary_axes", lambda: rotary_axes(dq, k, pos, [64])),
                 ("rotary_axes", lambda: rotary_axes(q, dk, pos, [64])), ("rotary_axes", lambda: rotary_axes(leaf, dk, pos, [64])),
                 ("sageattn_backward", lambda: sageattn_backward(dd, q, k, v, out, lse)),
                 ("sageattn_backward", lambda: sageattn_backward(dout, q, dk, v, out, lse))]
        for name, call in calls:
            with pytest.raises(NotImplementedError, match=name + ".*forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match=name + ".*forward-mode"):
                call()
        # over the backward pass: the gradient of the output carries the tangent
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(sageattn_train(leaf, k, v), leaf, dd)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(rotary_axes(leaf, None, pos, [64]), leaf, dd)
        plain = sageattn_train(q, k, v)
    assert torch.equal(plain, out)
