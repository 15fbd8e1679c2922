"""Rows whose scores are all huge (|score| of 10^8 to the type's range), in every kernel of ``sageattn``: equal scores
weigh alike, smaller ones not at all, and rows of ordinary scores in the same block are as ever.

Q and K hold the score in one channel, so equal scores are equal bits.  P is then 1 or 0 and the output the mean of V over
the keys of the largest score.  Tolerance: V to fp16 (2^-11 of it where it is not exact), up to 700 terms summed in fp32
(2^-14 of the mean of |V|), the output's own rounding; the LSE, score + ln n, is fp32 through five roundings (2^-22).  The
INT8 path's score passes the scales, fl(q fl(scale log2 e)) / 127 and k / 127, whose product loses its 3 lowest bits (up to
7 2^-23): with the 8 roundings of 2^-24 around it, 22 2^-24 in all."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
LOWEST = float(torch.finfo(BF16).min)
SCORES = [(F16, 65504.0, 65504.0), (F16, -65504.0, 30000.0), (BF16, 1.0, 1e9), (BF16, 1.0, 5e9), (BF16, 1.0, -1e10),
          (BF16, 1.0, 1e20), (BF16, -1.0, 1e20), (BF16, 1.0, LOWEST), (BF16, -1.0, LOWEST)]


def make(sq, sk, d, dtype, a, b, second=None):
    """q, k, v: every score a b / sqrt(d), or for the keys of every other 16 second times that."""
    g = torch.Generator().manual_seed(sq + sk)
    q, k, v = torch.zeros(1, 2, sq, d), torch.zeros(1, 2, sk, d), torch.randn(1, 2, sk, d, generator=g)
    q[..., 0] = a
    k[..., 0] = b
    top = torch.ones(sk, dtype=torch.bool)
    if second is not None:
        top[torch.arange(sk) // 16 % 2 == 0] = False
        k[:, :, ~top, 0] = b * second
    return [x.to(dtype).cuda() for x in (q, k, v)] + [top.cuda()]


def check(o, lse, q, k, v, weights, path="direct", scale=None):
    """weights [sq, sk]: 1 for the keys of a row's largest score, else 0."""
    w = weights.double()
    n = w.sum(-1, keepdim=True)
    want, size = w @ v.double() / n, w @ v.double().abs() / n
    off = (o.double() - want).abs()
    assert (off <= (torch.finfo(o.dtype).eps / 2 + 2.0 ** -20) * want.abs() + (2.0 ** -11 + 2.0 ** -14) * size).all(), off.max().item()
    s = (q.double()[..., :1] @ k.double()[..., :1].transpose(-1, -2)).masked_fill(w == 0, float("-inf")).amax(-1) * (scale or q.shape[-1] ** -0.5)
    want_lse = s + n[..., 0].log()
    assert ((lse.double() - want_lse).abs() <= (4 if path == "direct" else 22) * 2.0 ** -24 * want_lse.abs() + 1e-5).all()


def int8(monkeypatch, longest_direct=-1):
    for name in ("D64", "D64_CAUSAL", "D64_CROSS", "D128", "D128_CROSS"):
        monkeypatch.setenv("SAGEATTN_DIRECT_THRESHOLD_" + name, str(longest_direct))


@pytest.mark.parametrize("dtype,a,b", SCORES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("path", ["direct", "int8"])
@pytest.mark.parametrize("sq,sk,splits,causal", [(1, 416, 0, False), (90, 416, 1, False), (600, 416, 1, False), (600, 384, 3, False),
                                                 (600, 600, 0, True), (300, 300, 0, True)])
def test_equal_scores(dtype, a, b, d, path, sq, sk, splits, causal, monkeypatch):
    from sageattention import sageattn

    if path == "int8":
        int8(monkeypatch)
    if splits:
        monkeypatch.setenv("SAGEATTN_KV_SPLITS", str(splits))
    q, k, v, _ = make(sq, sk, d, dtype, a, b)
    o, lse = sageattn(q, k, v, is_causal=causal, return_lse=True)
    w = torch.ones(sq, sk, device="cuda")
    check(o, lse, q, k, v, w.tril() if causal else w, path)


@pytest.mark.parametrize("a,b", [(1.0, 1e9), (1.0, -1e10), (1.0, 1e20), (-1.0, LOWEST)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("path", ["direct", "int8"])
@pytest.mark.parametrize("sq,sk", [(1, 416), (600, 416)])
def test_two_scores(a, b, d, path, sq, sk, monkeypatch):
    """Half of the keys (in groups of 16, the first among them) score less by 2% or more: they do not count."""
    from sageattention import sageattn

    if path == "int8":
        int8(monkeypatch)
    q, k, v, top = make(sq, sk, d, BF16, a, b, 0.975 if a * b > 0 else 1.025)
    o, lse = sageattn(q, k, v, return_lse=True)
    check(o, lse, q, k, v, top.expand(sq, sk), path)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("path", ["direct", "int8"])
@pytest.mark.parametrize("sq,sk,causal", [(64, 500, False), (700, 500, False), (500, 500, True)])
def test_ordinary_rows_beside_huge_ones(d, path, sq, sk, causal, monkeypatch):
    """Every third 32 rows (a wave's) has a huge row; the others are those of a call without one, up to the rounding that
    another reference max brings (of P to fp16, 2^-11, and of sums)."""
    from sageattention import sageattn

    if path == "int8":
        int8(monkeypatch)
    g = torch.Generator().manual_seed(d + sq)
    q, k, v = (torch.randn(1, 2, s, d, generator=g) for s in (sq, sk, sk))
    q[..., 0] = 0
    k[..., 0] = 1e10
    rows = torch.arange(sq) % 96 == 5
    plain = q.to(BF16).cuda()
    q[:, :, rows] = 0
    # INT8 quantises 32 rows together: there the huge rows would take the others' bits, so they are whole groups
    if path == "int8":
        rows = torch.arange(sq) // 32 % 3 == 0
        q[:, :, rows] = 0
        k[..., 1:] = 0
        plain = plain * 0
        q = q * 0
    q[:, :, rows, 0] = 1
    q, k, v = (x.to(BF16).cuda() for x in (q, k, v))
    o, lse = sageattn(q, k, v, is_causal=causal, return_lse=True)
    want, want_lse = sageattn(plain, k, v, is_causal=causal, return_lse=True)
    keep = ~rows.cuda()
    size = sageattn(plain, k, v.abs(), is_causal=causal).double()
    assert ((o.double() - want.double()).abs()[:, :, keep] <= (2.0 ** -8 * want.double().abs() + 2.0 ** -9 * size)[:, :, keep]).all()
    assert ((lse - want_lse).abs()[:, :, keep] <= 1e-4).all()
    w = torch.ones(sq, sk, device="cuda")
    w = w.tril() if causal else w
    n = w.sum(-1, keepdim=True)
    huge = ((w @ v.float()) / n)[:, :, rows.cuda()]
    assert (o.float()[:, :, rows.cuda()] - huge).abs().max() <= 2.0 ** -8 * huge.abs().max() + 2.0 ** -9


@pytest.mark.parametrize("value", [-1e9, LOWEST])
@pytest.mark.parametrize("d", [64, 128])
def test_left_padded_causal(value, d):
    """Causal, the first keys masked by a large finite value: the output of the rows that see masked keys alone is the
    mean of those keys' V, in training's forward call too."""
    from sageattention import sageattn, sageattn_train

    pad, n = 70, 200
    q, k, v, _ = make(n, n, d, BF16, 1.0, 0.0)
    k[:, :, :pad, 0] = value
    w = torch.ones(pad, pad, device="cuda").tril()
    for o, lse in (sageattn(q, k, v, is_causal=True, return_lse=True),
                   sageattn_train(q.requires_grad_(True), k, v, is_causal=True, return_lse=True)):
        check(o[:, :, :pad].detach(), lse[:, :, :pad].detach(), q[:, :, :pad].detach(), k[:, :, :pad], v[:, :, :pad], w)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("order", ["low first", "high first", "mixed"])
@pytest.mark.parametrize("path", ["direct", "int8"])
@pytest.mark.parametrize("sq,d", [(1, 64), (600, 64), (600, 128)])
def test_scores_on_both_sides_of_the_line(sign, order, path, sq, d, monkeypatch):
    """Scores just below and just above 2^24 in log2 units, where a row's form changes (the two differ by thousands, so the
    larger ones have all the weight)."""
    from sageattention import sageattn

    if path == "int8":
        int8(monkeypatch)
    sk, values = 416, torch.tensor([1.155e7, 1.17e7]).to(BF16)
    assert values[0].item() * 1.4427 < 2 ** 24 < values[1].item() * 1.4427
    q, k, v, _ = make(sq, sk, d, BF16, 1.0, 0.0)
    i = torch.arange(sk)
    high = {"low first": i >= 208, "high first": i < 208, "mixed": i // 16 % 3 == 1}[order]
    k[..., 0] = torch.where(high, values[1], values[0]).cuda() * sign
    top = (high if sign > 0 else ~high).cuda()
    o, lse = sageattn(q, k, v, sm_scale=1.0, return_lse=True)
    w = top.expand(sq, sk)
    check(o, lse, q, k, v, w, path, 1.0)


@pytest.mark.parametrize("a,b", [(1.0, -1e9), (1.0, 5e9), (1.0, LOWEST)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("path", ["direct", "int8"])
@pytest.mark.parametrize("sq,sk,causal", [(200, 2300, False), (300, 4500, False), (2300, 2300, True), (130, 1100, False)])
def test_equal_scores_of_many_keys(a, b, d, path, sq, sk, causal, monkeypatch):
    """Many key tiles of a wave (the pipelined steps), two key groups of a block.  Unsplit: a split's LSE does not tell how
    many such keys it has.  bf16 V is exact in fp16, so the 2^-11 that `check` allows for it is there for the sums: 4500
    terms, 2^-11.8 of the mean of |V| at most."""
    from sageattention import sageattn

    int8(monkeypatch, -1 if path == "int8" else sk)
    monkeypatch.setenv("SAGEATTN_KV_SPLITS", "1")
    q, k, v, top = make(sq, sk, d, BF16, a, b, 0.975 if a * b > 0 else 1.025 if b > LOWEST else None)
    if causal:
        top[:] = True
        k[..., 0] = b
    o, lse = sageattn(q, k, v, is_causal=causal, return_lse=True)
    w = top.expand(sq, sk).float()
    check(o, lse, q, k, v, w.tril() if causal else w, path)
