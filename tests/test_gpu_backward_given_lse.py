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


def merged(q, k, v, dout, ranges, dtype, dlse=None, slack=0.0):
    """The gradients of attention over all keys from calls over the ranges, each with the whole output and LSE: dk and dv
    side by side, dq summed (each range's own rounded once more)."""
    from sageattention import sageattn_backward, sageattn_train

    out, lse = sageattn_train(q, k, v, return_lse=True)
    want, bounds = reference(q, k, v, dout, "HND", False, dlse=dlse)
    e = bounds(dtype)
    parts = [sageattn_backward(dout, q, k[:, :, r], v[:, :, r], out, lse, dlse=dlse) for r in ranges]
    for i, name in ((1, "dk"), (2, "dv")):
        check(torch.cat([p[i] for p in parts], 2), want[name], e[name], "HND", name)
    dq = [p[0].double() for p in parts]
    check(sum(dq), want["dq"], e["dq"] + torch.finfo(dtype).eps / 2 * sum(x.abs() for x in dq), "HND", "dq")


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (128, BF16)])
@pytest.mark.parametrize("dout_scale", [1.0, 64.0])
@pytest.mark.parametrize("small", [0.0, 1e-3])
@pytest.mark.parametrize("n", [64, 300])
def test_merged_ranges_of_unlike_values(d, dtype, dout_scale, small, n):
    """One range's V is far smaller than the other's, or zero (a padded block): delta is the merged output's, which that
    range's V does not bound."""
    q, k, v, dout = inputs(1, 2, 2, 150, 2 * n, d, dtype, "HND", seed=11, dout_scale=dout_scale)
    v[:, :, n:] *= small
    merged(q, k, v, dout, (slice(0, n), slice(n, 2 * n)), dtype)


@pytest.mark.parametrize("d", [64, 128])
def test_dead_rows_do_not_scale(d):
    """fp16 scales dS by the largest row of a kv head: a row without a live key has no dS and does not count, however
    large its gradients are."""
    from sageattention import sageattn, sageattn_backward

    q, k, v, dout = inputs(1, 2, 2, 100, 100, d, F16, "HND", dout_scale=1e-3)
    out, lse = sageattn(q, k, v, return_lse=True)
    dlse = torch.zeros_like(lse)
    lse[:, :, ::7] = float("-inf")
    dout[:, :, ::7] = 0
    want = sageattn_backward(dout, q, k, v, out, lse, dlse=dlse)
    dlse[:, :, ::7] = 1e30
    out[:, :, ::7] = 6e4
    dout[:, :, ::7] = 6e4
    for x, y in zip(sageattn_backward(dout, q, k, v, out, lse, dlse=dlse), want):
        assert torch.equal(x, y)
