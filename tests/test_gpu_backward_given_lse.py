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


def given(q, k, v, dout, out, lse, causal=False):
    """Gradients of the pass's own formula in 64 bits, P = min(1, exp(S - lse)) and delta = dout out from the given output
    and LSE, and their bounds.  Beside what ``reference`` counts, P is off by what the exponent is: S is summed in steps
    of 16 products of fp32 (2^-20 of the sum of |q||k| scale, with its factor's rounding), the LSE and its factor 2^-22;
    delta only by its own sum (2^-16 of the absolute one)."""
    q, k, v, dout, out = (x.double() for x in (q, k, v, dout, out))
    scale, g = q.shape[-1] ** -0.5, q.shape[1] // k.shape[1]
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = q @ kk.transpose(-1, -2) * scale
    if causal:
        s = s.masked_fill(torch.arange(s.shape[3], device=s.device) > torch.arange(s.shape[2], device=s.device)[:, None], float("-inf"))
    x = s - lse.double()[..., None]
    p = x.clamp(max=0).exp()
    dp, delta = dout @ vv.transpose(-1, -2), (dout * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)

    def fold(t):
        return t.reshape(t.shape[0], k.shape[1], g, *t.shape[2:]).sum(2)

    grads = dict(dq=ds @ kk * scale, dk=fold(ds.transpose(-1, -2) @ q) * scale, dv=fold(p.transpose(-1, -2) @ dout))

    def bounds(dtype):
        u, r = torch.finfo(dtype).eps / 2, 2.0 ** -16
        tiny = 2.0 ** -39 if dtype == F16 else 0.0
        r_p = 2.0 ** -20 * (q.abs() @ kk.abs().transpose(-1, -2)) * scale + 2.0 ** -22 * lse.double().abs()[..., None] + r
        bound = dout.norm(dim=-1).amax() * vv.norm(dim=-1).amax() + delta.abs().amax()
        sums = dout.abs() @ vv.abs().transpose(-1, -2) + (dout * out).abs().sum(-1, keepdim=True)
        e_p = (u + r_p) * p + tiny
        e_ds = (u + r_p) * ds.abs() + r * p * sums + tiny * bound
        e = dict(dq=e_ds @ kk.abs() * scale, dk=fold(e_ds.transpose(-1, -2) @ q.abs()) * scale,
                 dv=fold(e_p.transpose(-1, -2) @ dout.abs()))
        least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        return {n: e[n] + (u + r) * (grads[n].abs() + e[n]) + least for n in e}

    return grads, bounds, x


@pytest.mark.parametrize("d,dtype,causal,hq,hkv", [(128, F16, False, 2, 2), (128, F16, True, 4, 2), (64, F16, False, 2, 1),
                                                   (128, BF16, False, 2, 2), (64, BF16, True, 2, 2)])
@pytest.mark.parametrize("std,outlier", [(2.0, 16.0), (4.0, 4.0)])
def test_quantised_forward_with_an_outlier_channel(d, dtype, causal, hq, hkv, std, outlier, monkeypatch):
    """One channel of Q and K is far larger than the others, as in trained models: the INT8 path's rounding of the others
    then moves scores by whole units, and exp(score - LSE) is far above 1 for some pairs.  fp16 has no room for that."""
    from sageattention import sageattn, sageattn_backward

    for name in ("D64", "D64_CAUSAL", "D128"):
        monkeypatch.setenv("SAGEATTN_DIRECT_THRESHOLD_" + name, "-1")
    q, k, v, dout = inputs(1, hq, hkv, 2048, 2048, d, dtype, "HND")
    for x in (q, k):
        x *= std
        x[..., 7] *= outlier
    out, lse = sageattn(q, k, v, is_causal=causal, return_lse=True)
    want, bounds, x = given(q, k, v, dout, out, lse, causal)
    assert x.max() > 1.5, "no probability above 4"
    e = bounds(dtype)
    for name, got in zip(("dq", "dk", "dv"), sageattn_backward(dout, q, k, v, out, lse, is_causal=causal)):
        check(got, want[name], e[name], "HND", name)


def test_nan_lse_is_not_capped():
    """A row whose LSE is NaN (its scores are) has NaN gradients, not those of P = 1."""
    from sageattention import sageattn, sageattn_backward

    for dtype in (F16, BF16):
        q, k, v, dout = inputs(1, 1, 1, 90, 90, 64, dtype, "HND")
        out, lse = sageattn(q, k, v, return_lse=True)
        lse[0, 0, 40] = float("nan")
        dq, dk, dv = sageattn_backward(dout, q, k, v, out, lse)
        assert torch.isnan(dq[0, 0, 40]).all() and torch.isnan(dk).all() and torch.isnan(dv).all()
        assert torch.isfinite(dq[0, 0, :40]).all() and torch.isfinite(dq[0, 0, 41:]).all()


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16), (128, F16)])
@pytest.mark.parametrize("far", [40.0, 1000.0, 20000.0])
@pytest.mark.parametrize("n", [3, 20, 32])
def test_few_keys_of_a_merged_range(d, dtype, far, n):
    """A row's keys but for 2^-15 of its weight are a range of at most 32, whose P sum to 1 as nearly as fp32 tells.  The
    other keys' V is far larger: delta has to keep their part, which the range's own sum lacks."""
    q, k, v, dout = inputs(1, 2, 2, 150, n + 40, d, dtype, "HND", seed=12)
    q[..., 0], k[..., 0] = 1, 0
    k[:, :, n:] *= 0.25
    k[:, :, n:, 0] = -14.0 * d ** 0.5
    v[:, :, n:] *= far / 4
    merged(q, k, v, dout, (slice(0, n), slice(n, n + 40)), dtype)


@pytest.mark.parametrize("b,h,sq,sk,causal", [(1, 8, 64, 64, True), (1, 4, 131, 131, True), (2, 4, 200, 2, False), (1, 8, 300, 31, False)])
@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16), (64, BF16), (128, F16)])
def test_few_keys_of_a_whole_call(b, h, sq, sk, causal, d, dtype):
    """With the LSE of a call over these very keys, rows of few keys take delta from their probabilities as the autograd
    node does: the same bits."""
    from sageattention import sageattn_backward, sageattn_train

    q, k, v, dout = inputs(b, h, h, sq, sk, d, dtype, "HND", seed=8)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out, lse = sageattn_train(*leaves, is_causal=causal, return_lse=True)
    want = torch.autograd.grad(out, leaves, dout)
    got = sageattn_backward(dout, *(x.detach() for x in leaves), out.detach(), lse.detach(), is_causal=causal)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("seed", range(24))
def test_random_merges(seed):
    """Random range borders, scales of each range's K and V, shared heads, and a gradient of the LSE."""
    from sageattention import sageattn_backward, sageattn_train

    g = torch.Generator().manual_seed(100 + seed)

    def pick(*options):
        return options[torch.randint(len(options), (1,), generator=g).item()]

    d, dtype, group = pick(64, 128), pick(F16, BF16, F16), pick(1, 2, 4)
    hkv, sq = pick(1, 2, 3), pick(1, 31, 100, 300)
    sizes = [pick(1, 5, 32, 33, 100, 260) for _ in range(pick(2, 3))]
    q, k, v, dout = inputs(pick(1, 2), hkv * group, hkv, sq, sum(sizes), d, dtype, "HND", seed=seed, dout_scale=pick(1e-3, 1.0, 30.0))
    ranges, at = [], 0
    for n in sizes:
        r = slice(at, at + n)
        k[:, :, r] *= pick(0.1, 1.0, 2.0)
        v[:, :, r] *= pick(0.0, 1e-3, 1.0, 100.0)
        ranges.append(r)
        at += n
    out, lse = sageattn_train(q, k, v, return_lse=True)
    dlse = torch.randn(lse.shape, generator=g).cuda() * pick(0.0, 1.0, 1000.0)
    want, bounds = reference(q, k, v, dout, "HND", False, dlse=dlse)
    e = bounds(dtype)
    parts = [sageattn_backward(dout, q, k[:, :, r], v[:, :, r], out, lse, dlse=dlse) for r in ranges]
    for i, name in ((1, "dk"), (2, "dv")):
        check(torch.cat([p[i] for p in parts], 2), want[name], e[name], "HND", name)
    dq = [p[0].double() for p in parts]
    check(sum(dq), want["dq"], e["dq"] + torch.finfo(dtype).eps / 2 * sum(x.abs() for x in dq), "HND", "dq")


def test_captured_and_replayed():
    """The functional form in a graph, with smoothing and a NaN-free output, replayed with eager work between; two graphs
    of other sizes one after the other."""
    from sageattention import sageattn, sageattn_backward

    for s, dtype in ((2304, BF16), (2100, F16)):
        q, k, v, dout = inputs(1, 2, 1, s, s, 128, dtype, "HND")
        out, lse = sageattn(q, k, v, smooth_k=True, return_lse=True)
        ref = sageattn_backward(dout, q, k, v, out, lse, smooth_k=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            sageattn_backward(dout, q, k, v, out, lse, smooth_k=True)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = sageattn_backward(dout, q, k, v, out, lse, smooth_k=True)
        for _ in range(3):
            for x in got:
                x.zero_()
            graph.replay()
            torch.cuda.synchronize()
            again = sageattn_backward(dout, q, k, v, out, lse, smooth_k=True)
            assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(got, ref, again))
