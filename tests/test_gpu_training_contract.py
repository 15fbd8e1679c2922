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


@pytest.mark.parametrize("shape_q,shape_k", [((1, 1, 2 ** 24 - 127, 128), (1, 1, 64, 128)), ((1, 1, 64, 128), (1, 1, 2 ** 24, 128)),
                                             ((1, 1, 2 ** 25, 64), (1, 1, 64, 64)), ((4, 2 ** 14, 2 ** 15, 64), (4, 2 ** 14, 64, 64)),
                                             ((2 ** 24, 1, 64, 64), (2 ** 24, 1, 64, 64)), ((1, 1, 2 ** 31, 64), (1, 1, 64, 64))])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_limits_are_told_by_the_forward_call(shape_q, shape_k, layout):
    """Sizes that the backward pass does not take.  (Expanded tensors: no memory, and no kernel reads them.)"""
    from sageattention import sageattn_train
    from sageattention._capi import SageError

    def make(shape):
        x = torch.zeros(1, 1, 1, shape[3], dtype=BF16, device="cuda").requires_grad_(True).expand(shape)
        return x.transpose(1, 2) if layout == "NHD" else x

    q, k = make(shape_q), make(shape_k)
    before = torch.cuda.memory_allocated()
    with pytest.raises((SageError, ValueError), match="limits|tokens"):
        sageattn_train(q, k, k, tensor_layout=layout)
    assert torch.cuda.memory_allocated() == before


def test_many_heads_of_many_tokens():
    """[B,N,H,D] whose heads span more than 32-bit offsets, in q, the output and their gradients: the gradients of the
    same call head by head, bit for bit."""
    from sageattention import sageattn_train

    b, h, n, d = 1, 64, 262144, 128
    g = torch.Generator(device="cuda").manual_seed(2)
    q, dout = (torch.randn(b, n, h, d, generator=g, device="cuda", dtype=BF16) for _ in range(2))
    k, v = (torch.randn(b, 50, h, d, generator=g, device="cuda", dtype=BF16) for _ in range(2))

    def grads(layout):
        turn = (lambda x: x) if layout == "NHD" else (lambda x: x.transpose(1, 2).contiguous())
        leaves = [turn(x).requires_grad_(True) for x in (q, k, v)]
        out = sageattn_train(*leaves, tensor_layout=layout)
        return [x if layout == "NHD" else x.transpose(1, 2) for x in (out.detach(), *torch.autograd.grad(out, leaves, turn(dout)))]

    for x, y in zip(grads("NHD"), grads("HND")):
        assert x.shape == y.shape and torch.equal(x, y)


def one_token_slices(heads, d, dtype, layout, odd):
    """q, k, v and an output gradient of one token: slices of rows whose length is odd, so that the strides of the batch
    and token dimensions, of one element each, are odd too."""
    g = torch.Generator().manual_seed(4)
    row = torch.nn.functional.pad(torch.randn(1, 1, 4 * heads * d, generator=g), (0, odd)).to(dtype).cuda()
    out = [row[..., i * heads * d:(i + 1) * heads * d].reshape(1, 1, heads, d) if not odd else
           row[..., i * heads * d:(i + 1) * heads * d].as_strided((1, 1, heads, d), (row.shape[2], row.shape[2], d, 1), i * heads * d)
           for i in range(4)]
    return [x if layout == "NHD" else x.transpose(1, 2) for x in out]


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("odd", [1, 4])
def test_odd_strides_of_dimensions_of_one(layout, odd):
    from sageattention import rotary_axes, sageattn, sageattn_backward, sageattn_train

    def results(odd):
        q, k, v, dout = one_token_slices(4, 64, BF16, layout, odd)
        pos = torch.full((1, 1), 7, device="cuda")
        outs = list(rotary_axes(q, k, pos, [64], tensor_layout=layout))
        even = q.clone(memory_format=torch.contiguous_format)  # sageattn refuses odd strides of q, as the reference does
        outs.append(sageattn(even, k, v, tensor_layout=layout))
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out, lse = sageattn_train(*leaves, tensor_layout=layout, return_lse=True)
        outs += [out.detach(), lse.detach(), *torch.autograd.grad(out, leaves, dout)]
        outs += sageattn_backward(dout, q, k, v, out.detach(), lse.detach(), tensor_layout=layout)
        return outs

    for x, y in zip(results(odd), results(0)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("frozen", ["q", "k"])
def test_rotary_of_an_input_without_gradient(frozen):
    """The turned q or k of an input that needs no gradient needs none itself; the other's gradient is the same."""
    from sageattention import rotary_axes

    q, k, _, _ = inputs(1, 4, 2, 50, 50, 64, F32, "HND")
    pos = torch.arange(50, device="cuda")[:, None]
    both = [x.clone().requires_grad_(True) for x in (q, k)]
    outs = rotary_axes(*both, pos, [64])
    weights = [torch.randn_like(x) for x in outs]
    want = torch.autograd.grad(outs, both, weights, create_graph=True)
    assert all(x.requires_grad for x in outs)
    one = [x.clone().requires_grad_(name != frozen) for name, x in (("q", q), ("k", k))]
    turned = rotary_axes(*one, pos, [64])
    assert [x.requires_grad for x in turned] == [frozen != "q", frozen != "k"]
    i = 1 if frozen == "q" else 0
    got = torch.autograd.grad(turned[i], one[i], weights[i])[0]
    assert torch.equal(got, want[i]) and torch.equal(turned[i], outs[i]) and torch.equal(turned[1 - i], outs[1 - i])


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_rows_far_apart(layout):
    """Two tokens 32 MB apart in q, v and the output's gradient: past the kernels' 32-bit offsets (which run 128 rows past
    the end), so they are copied."""
    from sageattention import sageattn_train

    g = torch.Generator().manual_seed(6)
    near = [torch.randn(1, 3, 2, 64, generator=g).to(BF16).cuda() for _ in range(4)]
    far = []
    for x in near:
        y = torch.zeros(2 ** 24 + 3 * 64, dtype=BF16, device="cuda").as_strided((1, 3, 2, 64), (2 ** 25, 64, 2 ** 24, 1))
        y.copy_(x)
        far.append(y)
    far[1] = near[1]  # the forward call refuses such a k

    def grads(tensors):
        q, k, v, dout = (x if layout == "HND" else x.transpose(1, 2) for x in tensors)
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = sageattn_train(*leaves, tensor_layout=layout)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    for x, y in zip(grads(far), grads(near)):
        assert torch.equal(x, y)
