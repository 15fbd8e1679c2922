"""Performance cases of the training operators: attention with its gradient, and rotary positions over several axes.

Programs that train (or fine-tune) image, video and language models call ``rotary_axes`` on the queries and keys of a
layer, with a token's position on each axis (time, height, width), then ``sageattn_train``, and later run the backward
pass of both.  A pass here is what one layer of such a step does with the operator: forward and gradients through
autograd for ``sageattn_train``; forward, or forward and gradients, for ``rotary_axes``.

``own`` false computes the same outputs in plain elementary operations.
"""
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _own():
    import os
    import sys

    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sageattention-rdna3_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import sageattention

    return sageattention


def _attn(name, b, hq, hkv, sq, sk, d, dtype, layout, causal=False):
    c = dict(op="attn", b=b, hq=hq, hkv=hkv, sq=sq, sk=sk, d=d, dtype=dtype, layout=layout, causal=causal)
    return dict(c, name=name) if name else c


def _rotary(name, b, hq, hkv, text, t, h, w, d, axes, dtype, layout, interleaved=True, grad=False, fractional=False):
    """`text` tokens at the origin, then a grid of t x h x w tokens."""
    c = dict(op="rotary", b=b, hq=hq, hkv=hkv, text=text, t=t, h=h, w=w, d=d, axes=axes, dtype=dtype, layout=layout,
             interleaved=interleaved, grad=grad, fractional=fractional)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a deep block of a small image: the smallest training call, where launches count
        _attn("attn_small", 1, 10, 10, 256, 256, 64, "fp16", "NHD"),
        # image tokens attending 77 text tokens (few keys, many queries)
        _attn("attn_text_cross", 2, 10, 10, 4096, 77, 64, "fp16", "NHD"),
        # image tokens attending 512 conditioning tokens
        _attn("attn_cond_cross", 1, 16, 16, 4096, 512, 128, "bf16", "NHD"),
        # image self-attention at head_dim 64
        _attn("attn_self_d64", 1, 10, 10, 4096, 4096, 64, "fp16", "HND"),
        # a ragged mid-length sequence of few heads, in the layout projections give
        _attn("attn_ragged", 1, 12, 12, 2393, 2393, 128, "bf16", "NHD"),
        # language-model training on a batch of short texts, grouped heads
        _attn("attn_causal_gqa", 2, 32, 8, 2048, 2048, 128, "bf16", "NHD", causal=True),
        # the largest: a long video or image sequence
        _attn("attn_self_long", 1, 24, 24, 8192, 8192, 128, "bf16", "HND"),
        # one small image's queries and keys at inference: latency
        _rotary("rotary_small", 1, 10, 10, 0, 1, 16, 16, 64, "32,32", "fp16", "NHD"),
        # an image with its text tokens in one sequence, forward and gradients
        _rotary("rotary_image", 1, 16, 16, 512, 1, 64, 64, 128, "16,56,56", "bf16", "HND", grad=True),
        # a grouped-head model that pairs the halves of the head, in float32, odd sizes
        _rotary("rotary_halves", 2, 28, 4, 77, 5, 31, 27, 128, "32,48,48", "fp32", "NHD", interleaved=False, grad=True),
        # a long video: the largest
        _rotary("rotary_video", 1, 40, 40, 0, 21, 36, 43, 128, "44,42,42", "bf16", "HND"),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]; one in three a multiple of 64 where that fits."""
    n = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 1 / 3 and n >= 64:
        n = n // 64 * 64
    return max(lo, min(hi, n))


def draw(rng):
    d = rng.choice([64, 128])
    dtype = rng.choice(["fp16", "bf16"])
    layout = rng.choice(["HND", "NHD"])
    kind = rng.choice(["cross", "self", "causal", "self", "rotary", "rotary"])
    if kind == "rotary":
        axes = rng.choice(["32,32", "16,24,24", "20,22,22", "8,16,16", "64"] if d == 64 else
                          ["16,56,56", "44,42,42", "32,48,48", "64,64", "16,40,40", "128"])
        n_axes = axes.count(",") + 1
        text = rng.choice([0, 77, rng.randint(1, 512)])
        t = 1 if n_axes < 3 else rng.randint(1, 16)
        h, w = (1, _log(rng, 1, 8192)) if n_axes == 1 else (rng.randint(4, 56), rng.randint(4, 56))
        hkv = rng.choice([4, 8, 10, 16])
        group = rng.choice([1, 1, 2, 4]) if hkv <= 8 else 1
        b = rng.choice([1, 1, 2])
        while b * hkv * (group + 1) * (text + t * h * w) > 2 * 40 * 32508 / 2:  # gradients move twice the bytes
            t = max(1, t // 2)
            h = max(1, h - 4)
            b = 1
        return _rotary(None, b, hkv * group, hkv, text, t, h, w, d, axes, rng.choice([dtype, dtype, "fp32"]), layout,
                       interleaved=rng.random() < 0.6, grad=rng.random() < 0.5, fractional=rng.random() < 0.25)
    h = rng.choice([5, 8, 10, 16, 24])
    group = rng.choice([1, 1, 1, 2, 4])
    b = rng.choice([1, 1, 2])
    limit = 24 * 8192 * 8192  # scores of the largest listed case
    if kind == "cross":
        sq, sk = _log(rng, 64, 9216), _log(rng, 16, 1024)
    elif kind == "self":
        sq = sk = _log(rng, 64, 8192)
    else:
        sq = sk = _log(rng, 64, 4096)
    if b * h * group * sq * sk > limit:
        b = group = 1
    return _attn(None, b, h * group, h, sq, sk, d, dtype, layout, causal=kind == "causal")


def _normal(g, case, heads, tokens):
    b, d = case["b"], case["d"]
    shape = (b, tokens, heads, d) if case["layout"] == "NHD" else (b, heads, tokens, d)
    return torch.randn(shape, generator=g, device="cuda")


def _positions(case, g):
    """[N, axes]: text tokens at the origin, then the grid; a case of fractional positions shifts and scales the grid
    (resolution other than the one trained at)."""
    sizes = [case["t"], case["h"], case["w"]]
    sizes = sizes[-(case["axes"].count(",") + 1):]
    grid = torch.cartesian_prod(*[torch.arange(n, device="cuda") for n in sizes]).reshape(-1, len(sizes))
    pos = torch.cat([torch.zeros(case["text"], len(sizes), dtype=grid.dtype, device="cuda"), grid])
    if case["fractional"]:
        pos = pos.float() * 0.71 + torch.rand(len(sizes), generator=g, device="cuda")
    return pos


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "attn":
        q = _normal(g, case, case["hq"], case["sq"])
        k, v = _normal(g, case, case["hkv"], case["sk"]), _normal(g, case, case["hkv"], case["sk"])
        # fp16 training scales its loss, bf16 training does not
        dout = _normal(g, case, case["hq"], case["sq"]) * (1.0 if case["dtype"] == "fp16" else 1e-3)
        return tuple(x.to(dt) for x in (q, k, v, dout))
    n = case["text"] + case["t"] * case["h"] * case["w"]
    q, k = _normal(g, case, case["hq"], n).to(dt), _normal(g, case, case["hkv"], n).to(dt)
    dq = dk = None
    if case["grad"]:
        dq, dk = _normal(g, case, case["hq"], n).to(dt), _normal(g, case, case["hkv"], n).to(dt)
    return q, k, dq, dk, _positions(case, g)


def prepare(case, seed):
    inputs = _inputs(case, seed)
    leaves = inputs[:3] if case["op"] == "attn" else inputs[:2] if case["grad"] else ()
    for x in leaves:
        x.requires_grad_(True)
    return (case,) + inputs


def _heads_first(x, case):
    return x.transpose(1, 2) if case["layout"] == "NHD" else x


def _plain_attn(case, q, k, v, dout):
    """Softmax attention and its gradients with the whole score matrix in float32."""
    dt, scale = q.dtype, case["d"] ** -0.5
    b, hkv, sk, d = case["b"], case["hkv"], case["sk"], case["d"]
    rows = case["hq"] // hkv, case["sq"]

    def grouped(x):  # [b, hkv, group, s, d]
        return _heads_first(x, case).float().reshape(b, hkv, *rows, d)

    q, dout = grouped(q), grouped(dout)
    k, v = (_heads_first(x, case).float().unsqueeze(2).contiguous() for x in (k, v))
    k_t, v_t = k.transpose(-1, -2).contiguous(), v.transpose(-1, -2).contiguous()
    p = (q * scale) @ k_t
    if case["causal"]:
        future = torch.arange(sk, device="cuda") > torch.arange(case["sq"], device="cuda")[:, None]
        p.masked_fill_(future, float("-inf"))
    p -= p.amax(-1, keepdim=True)
    p.exp_()
    p /= p.sum(-1, keepdim=True)
    out = p @ v
    dv = (p.transpose(-1, -2) @ dout).sum(2)
    ds = dout @ v_t
    ds -= (dout * out).sum(-1, keepdim=True)
    ds *= p
    del p
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2) * scale
    flat = [x.reshape(b, -1, rows[1], d) for x in (out, dq)] + [dk, dv]
    return tuple(_heads_first(x, case).to(dt).contiguous() for x in flat)


def _angles(case, positions):
    """[N, R/2] in float64: pair j of an axis of width d turns by position * theta^(-2j/d)."""
    parts = []
    for a, width in enumerate(int(x) for x in case["axes"].split(",")):
        freq = 10000.0 ** (-torch.arange(0, width, 2, dtype=torch.float64, device="cuda") / width)
        parts.append(positions[:, a].double()[:, None] * freq)
    return torch.cat(parts, 1)


def _plain_rotate(case, x, cos, sin, sign):
    pairs = cos.shape[-1]
    if case["layout"] == "NHD":
        cos, sin = cos[:, None], sin[:, None]
    y = x.float()
    out = y.clone()
    first, second = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if case["interleaved"] else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = y[..., first], y[..., second]
    out[..., first] = a * cos - b * sin * sign
    out[..., second] = b * cos + a * sin * sign
    return out.to(x.dtype)


def run(state):
    case, inputs = state[0], state[1:]
    if case["op"] == "attn":
        q, k, v, dout = inputs
        if own:
            out = _own().sageattn_train(q, k, v, tensor_layout=case["layout"], is_causal=case["causal"])
            return (out.detach(),) + torch.autograd.grad(out, (q, k, v), dout)
        with torch.no_grad():
            return _plain_attn(case, q, k, v, dout)
    q, k, dq, dk, positions = inputs
    if own:
        axes = [int(x) for x in case["axes"].split(",")]
        outs = _own().rotary_axes(q, k, positions, axes, tensor_layout=case["layout"], interleaved=case["interleaved"])
        grads = torch.autograd.grad(outs, (q, k), (dq, dk)) if case["grad"] else ()
        return tuple(x.detach() for x in outs) + tuple(grads)
    with torch.no_grad():
        angle = _angles(case, positions)
        cos, sin = angle.cos().float(), angle.sin().float()
        outs = (_plain_rotate(case, q, cos, sin, 1.0), _plain_rotate(case, k, cos, sin, 1.0))
        if case["grad"]:
            outs += (_plain_rotate(case, dq, cos, sin, -1.0), _plain_rotate(case, dk, cos, sin, -1.0))
        return outs


def work(case):
    e = DTYPES[case["dtype"]].itemsize
    b, hq, hkv, d = (case[n] for n in ("b", "hq", "hkv", "d"))
    if case["op"] == "attn":
        sq, sk = case["sq"], case["sk"]
        pairs = sq * sk
        if case["causal"]:  # top-left mask: row i sees keys 0..i
            n = min(sq, sk)
            pairs = n * (n + 1) // 2 + (sq - n) * sk
        # in: q, k, v, dout; out: out, dq, dk, dv; products: two forward, five backward
        return {"bytes": e * d * b * (4 * hq * sq + 4 * hkv * sk), "flops": 14 * b * hq * d * pairs}
    n = case["text"] + case["t"] * case["h"] * case["w"]
    passes = 2 if case["grad"] else 1
    moved = 2 * e * d * b * (hq + hkv) * n
    position = n * (case["axes"].count(",") + 1) * (4 if case["fractional"] else 8)
    return {"bytes": passes * moved + position, "flops": passes * 3 * d * b * (hq + hkv) * n}


def _exact_attn(case, seed):
    """Head by head and in pieces of rows, from the definition in 64 bits."""
    q, k, v, dout = (_heads_first(x, case).double() for x in _inputs(case, seed))
    scale, group = case["d"] ** -0.5, case["hq"] // case["hkv"]
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i in range(case["b"]):
        for h in range(case["hq"]):
            j = h // group
            for r in range(0, case["sq"], 4096):
                rows = torch.arange(r, min(case["sq"], r + 4096), device="cuda")
                s = torch.mm(q[i, h, rows], k[i, j].T.contiguous()) * scale
                if case["causal"]:
                    s[torch.arange(case["sk"], device="cuda")[None] > rows[:, None]] = float("-inf")
                p = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
                g = dout[i, h, rows]
                out[i, h, rows] = torch.mm(p, v[i, j])
                dp = torch.mm(g, v[i, j].T.contiguous())
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                dq[i, h, rows] = torch.mm(ds, k[i, j])
                dk[i, j] += torch.mm(ds.T.contiguous(), q[i, h, rows])
                dv[i, j] += torch.mm(p.T.contiguous(), g)
    return tuple(_heads_first(x, case).contiguous() for x in (out, dq, dk, dv))


def _exact_rotary(case, seed):
    """A pair as a complex number times exp(i angle), in 64 bits."""
    q, k, dq, dk, positions = _inputs(case, seed)
    widths = [int(x) for x in case["axes"].split(",")]
    total = sum(widths)
    turn = torch.empty(positions.shape[0], total // 2, dtype=torch.complex128, device="cuda")
    at = 0
    for a, width in enumerate(widths):
        j = torch.arange(width // 2, dtype=torch.float64, device="cuda")
        angle = positions[:, a, None].double() / torch.pow(torch.tensor(10000.0, dtype=torch.float64, device="cuda"), 2 * j / width)
        turn[:, at:at + width // 2] = torch.polar(torch.ones_like(angle), angle)
        at += width // 2

    def rotated(x, w):
        y = _heads_first(x, case).double()
        head, rest = y[..., :total], y[..., total:]
        pair = head.unflatten(-1, (total // 2, 2)) if case["interleaved"] else head.unflatten(-1, (2, total // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * w)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        return _heads_first(torch.cat([z.flatten(-2), rest], -1), case).contiguous()

    outs = (rotated(q, turn), rotated(k, turn))
    return outs + ((rotated(dq, turn.conj()), rotated(dk, turn.conj())) if case["grad"] else ())


def exact(case, seed):
    with torch.no_grad():
        return _exact_attn(case, seed) if case["op"] == "attn" else _exact_rotary(case, seed)
