"""``sageattn_backward`` with an output and LSE that are not those of one call of the direct kernel over these keys: the
INT8 path's (with and without K smoothing), or those of several key ranges merged."""
import pytest
import torch

from _training import check, heads_first, inputs, reference

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("d,dtype,layout,causal,s", [(128, BF16, "HND", False, 2500), (128, F16, "NHD", True, 2500), (64, BF16, "NHD", False, 3200)])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (4, 2)])
def test_smoothed_forward(d, dtype, layout, causal, s, hq, hkv):
    """K with an offset per channel, which smoothing takes out.  What is left is the path's rounding of Q and K - mean to 8
    bits, as without an offset: a few per cent (a tenth at most); with the LSE taken as that of K itself the
    probabilities of a row are off by exp(scale q.mean), the exponent of deviation 2 here."""
    from sageattention import sageattn, sageattn_backward

    q, k, v, dout = inputs(1, hq, hkv, s, s, d, dtype, layout)
    offset = torch.randn(1, 1, hkv, d, generator=torch.Generator().manual_seed(3)) * 2
    offset = offset if layout == "NHD" else offset.transpose(1, 2)
    k = (k.float() + offset.cuda()).to(dtype)
    out, lse = sageattn(q, k, v, tensor_layout=layout, is_causal=causal, smooth_k=True, return_lse=True)
    want, _ = reference(q, k, v, dout, layout, causal)
    assert (lse.double() - want["lse"]).abs().max() > 1, "the call did not smooth"
    got = sageattn_backward(dout, q, k, v, out, lse, tensor_layout=layout, is_causal=causal, smooth_k=True)
    for name, x in zip(("dq", "dk", "dv"), got):
        off = (heads_first(x, layout).double() - want[name]).norm() / want[name].norm()
        assert off < 0.1, (name, off.item())


def test_smoothing_of_a_direct_call_is_none(monkeypatch):
    """Short calls take the direct kernel, whatever smooth_k: so does their backward pass, with the dispatch's overrides."""
    from sageattention import sageattn, sageattn_backward

    q, k, v, dout = inputs(1, 2, 2, 300, 300, 128, BF16, "HND")
    k = k + 3
    out, lse = sageattn(q, k, v, smooth_k=True, return_lse=True)
    dlse = torch.ones_like(lse)
    a = sageattn_backward(dout, q, k, v, out, lse, smooth_k=True, dlse=dlse)
    assert all(torch.equal(x, y) for x, y in zip(a, sageattn_backward(dout, q, k, v, out, lse, dlse=dlse)))
    want, bounds = reference(q, k, v, dout, "HND", False, dlse=dlse)
    for name, x in zip(("dq", "dk", "dv"), a):
        check(x, want[name], bounds(BF16)[name], "HND", name)
    monkeypatch.setenv("SAGEATTN_DIRECT_THRESHOLD_D128", "-1")
    out, lse = sageattn(q, k, v, smooth_k=True, return_lse=True)
    want, _ = reference(q, k, v, dout, "HND", False)
    for name, x in zip(("dq", "dk", "dv"), sageattn_backward(dout, q, k, v, out, lse, smooth_k=True)):
        assert (x.double() - want[name]).norm() < 0.1 * want[name].norm(), name
    with pytest.raises(ValueError, match="dlse"):
        sageattn_backward(dout, q, k, v, out, lse, smooth_k=True, dlse=dlse)


def test_smoothed_empty():
    from sageattention import sageattn_backward

    for b, sq, sk in ((0, 3000, 3000), (1, 0, 3000)):
        q, k, v, dout = inputs(b, 2, 2, sq, sk, 128, BF16, "HND")
        lse = torch.zeros(b, 2, sq, device="cuda")
        got = sageattn_backward(dout, q, k, v, q, lse, smooth_k=True)
        assert [x.shape for x in got] == [q.shape, k.shape, v.shape] and not any(x.any() for x in got)
