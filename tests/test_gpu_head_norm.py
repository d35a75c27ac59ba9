"""Head norms with the position rotation (qk_norm_rope, qk_norm_rope_backward) against the formulas in 64 bits.

Bounds, in units of 2^-24 of a pair's |u_1| + |u_2|: the sum of squares is a chain of at most 16 roundings in a lane and 6 over
the lanes, halved by the root, the root itself 2, three products 3, the angle (an argument and a series below pi / 4) 4, the
turn 3: 24 in all.  The gradient goes through one more such sum: 48 of the largest terms.  Then eps / 2 of the result's type."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a device"
    from proteinpredictmachinelearning_amd import ops as _ops

    return _ops


def pairs_of(rot, interleaved):
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def turned(u, freqs, positions, interleaved, sign=1.0):
    """(R(p) u, |u_1| + |u_2| of each element's pair) for u (B, L, h, d) in 64 bits on the CPU"""
    size = u.abs().clone()
    if freqs is None or freqs.numel() == 0:
        return u.clone(), size
    one, two = pairs_of(2 * freqs.numel(), interleaved)
    angle = (positions.double().unsqueeze(-1) * freqs.double().cpu()).unsqueeze(2)
    c, s = torch.cos(angle), sign * torch.sin(angle)
    y = u.clone()
    y[..., one], y[..., two] = u[..., one] * c - u[..., two] * s, u[..., two] * c + u[..., one] * s
    size[..., one] = size[..., two] = u[..., one].abs() + u[..., two].abs()
    return y, size


def all_positions(positions, B, L):
    if positions is None:
        return torch.arange(L).expand(B, L)
    return positions.cpu().expand(B, L)


def forward(x, w, freqs, positions, eps, interleaved):
    x = x.double().cpu()
    u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        u = u * w.double().cpu()
    y, size = turned(u, freqs, all_positions(positions, x.shape[0], x.shape[1]), interleaved)
    return y.transpose(1, 2), size.transpose(1, 2)


def backward(dy, x, w, freqs, positions, eps, interleaved):
    """(dx, its bound, dw, its bound) in 64 bits"""
    x = x.double().cpu()
    v, size = turned(dy.double().cpu().transpose(1, 2), freqs, all_positions(positions, x.shape[0], x.shape[1]), interleaved, sign=-1.0)
    s = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    n = x * s
    dw = (v * n).sum((0, 1, 2))
    # a sum's own error: of each of its terms as many roundings as a chain of the kernels has at most, 128 here
    dw_bound = (48 + 128) * UNIT * (size * n.abs()).sum((0, 1, 2))
    scale = torch.ones(()) if w is None else w.double().cpu()
    g = v * scale
    gs = size * scale.abs()
    dx = s * (g - n * (g * n).mean(-1, keepdim=True))
    bound = 48 * UNIT * s * (gs + n.abs() * (gs * n.abs()).mean(-1, keepdim=True))
    return dx, bound, dw, dw_bound


def close(got, want, bound):
    half = torch.finfo(got.dtype).eps / 2
    bound = 1.01 * (bound + half * (want.abs() + bound)) + torch.finfo(got.dtype).smallest_normal * half
    err = (got.double().cpu() - want).abs()
    assert (err <= bound).all(), f"largest excess {(err - bound).max().item():.3e}, value {want.abs().max().item():.3e}"


# B, L, hq, hk, d, rot, interleaved
CASES = [
    (1, 1, 1, 1, 2, 2, False),          # the smallest head that turns
    (1, 1, 1, 1, 1, 0, False),          # one element, nothing turns
    (1, 1, 8, 8, 32, 32, False),        # one token
    (2, 51, 8, 8, 32, 32, False),       # an alignment's rows
    (1, 103, 4, 4, 32, 16, True),
    (3, 17, 8, 2, 128, 128, False),     # shared key heads
    (1, 37, 32, 8, 128, 64, True),
    (2, 9, 3, 1, 64, 0, False),
    (1, 33, 5, 3, 80, 80, False),
    (1, 20, 4, 4, 24, 24, False),
    (2, 11, 2, 2, 24, 24, True),
    (1, 13, 4, 2, 7, 6, False),         # odd heads: one element at a time
    (1, 13, 4, 2, 31, 10, True),
    (1, 19, 2, 3, 66, 66, False),
    (1, 5, 2, 2, 130, 12, False),
    (1, 6, 2, 1, 257, 256, True),
    (1, 4, 2, 2, 512, 512, False),      # the widest
    (1, 4, 1, 1, 511, 510, False),
    (2, 3, 2, 2, 256, 192, False),
    (1, 700, 2, 2, 16, 8, False),
    (1, 16400, 2, 1, 64, 64, False),    # sixteen-bit types eight elements at a time
    (1, 33000, 1, 1, 48, 16, False),
    (2, 8300, 1, 2, 64, 32, True),
    (1, 3000, 2, 1, 8, 8, False),       # work-groups of the backward pass that take several tokens each
]


def operands(B, L, hq, hk, d, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(B, L, (hq + 2 * hk) * d, device="cuda", generator=gen) * torch.exp(torch.randn(B, L, 1, device="cuda", generator=gen))).to(dtype)
    q, k = qkv[..., :hq * d].unflatten(-1, (hq, d)), qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    wq, wk = (1 + 0.3 * torch.randn(d, device="cuda", generator=gen) for _ in range(2))
    dq, dk = (torch.randn(B, h, L, d, device="cuda", generator=gen).to(dtype) for h in (hq, hk))
    return q, k, wq, wk, dq, dk, gen


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,hq,hk,d,rot,interleaved", CASES)
def test_forward_and_backward_match_the_formulas(ops, B, L, hq, hk, d, rot, interleaved, dtype):
    q, k, wq, wk, dq, dk, gen = operands(B, L, hq, hk, d, dtype, 100 * d + L)
    freqs = ops.rope_frequencies(rot) if rot else None
    positions = torch.randint(0, 4000, (B, L), device="cuda", generator=gen, dtype=torch.int32) if L % 2 else None
    kw = dict(eps=1e-6, interleaved=interleaved)
    yq, yk = ops.qk_norm_rope(q, k, wq, wk, freqs, positions, **kw)
    assert yq.is_contiguous() and yk.is_contiguous() and yq.dtype == dtype
    for y, x, w in ((yq, q, wq), (yk, k, wk)):
        want, size = forward(x, w, freqs, positions, 1e-6, interleaved)
        close(y, want, 24 * UNIT * size)
    gq, gk, gwq, gwk = ops.qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs, positions, **kw)
    for g, gw, dy, x, w in ((gq, gwq, dq, q, wq), (gk, gwk, dk, k, wk)):
        dx, bound, dw, dw_bound = backward(dy, x, w, freqs, positions, 1e-6, interleaved)
        close(g, dx, bound)
        close(gw, dw, dw_bound)


@pytest.mark.parametrize("d,rot,interleaved", [(32, 32, False), (16, 8, True), (7, 4, False)])
def test_gradients_match_differences(ops, d, rot, interleaved):
    """Central differences of the 64-bit formula in some directions: a formula's mistake would show here"""
    q, k, wq, wk, dq, dk, gen = operands(1, 5, 2, 1, d, torch.float32, d)
    freqs = ops.rope_frequencies(rot)
    grads = ops.qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs, None, interleaved=interleaved)
    inputs = [t.double().cpu() for t in (q, k, wq, wk)]

    def loss(q, k, wq, wk):
        return sum((forward(x, w, freqs, None, 1e-6, interleaved)[0] * dy.double().cpu()).sum() for x, w, dy in ((q, wq, dq), (k, wk, dk)))

    for i in range(4):
        for _ in range(3):
            direction = torch.randn(inputs[i].shape, dtype=torch.float64)
            step = 1e-5
            moved = [[t + s * step * direction if j == i else t for j, t in enumerate(inputs)] for s in (1, -1)]
            slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
            along = (grads[i].double().cpu() * direction).sum()
            # (the differences' own error is below 1e-8 of these sizes, the gradient's as above)
            assert abs(slope - along) <= 1e-5 * (grads[i].double().cpu() * direction).abs().sum()


@pytest.mark.parametrize("kind", ["no_weights", "only_q", "shared_positions", "int64", "negative", "far"])
def test_options(ops, kind):
    B, L, hq, hk, d = 2, 23, 4, 2, 32
    q, k, wq, wk, dq, dk, gen = operands(B, L, hq, hk, d, torch.float32, 9)
    freqs, positions = ops.rope_frequencies(d, base=500.0), None
    if kind == "no_weights":
        wq = wk = None
    if kind == "only_q":
        wk = None
    if kind == "shared_positions":
        positions = torch.randint(0, 1000, (L,), device="cuda", generator=gen, dtype=torch.int32)
    if kind == "int64":
        positions = torch.randint(0, 1 << 40, (B, L), device="cuda", generator=gen)
        freqs = freqs * 2.0 ** -20
    if kind == "negative":
        positions = torch.randint(-5000, 0, (B, L), device="cuda", generator=gen, dtype=torch.int32)
    if kind == "far":
        positions = torch.randint(10 ** 9, 2 ** 31 - 1, (B, L), device="cuda", generator=gen, dtype=torch.int32)
    # an angle p f in 64 bits is off by 2^-53 of itself in the kernel (twice) and in the test
    loose = 0.0 if positions is None else float(positions.abs().max()) * float(freqs.max()) * 2.0 ** -51
    yq, yk = ops.qk_norm_rope(q, k, wq, wk, freqs, positions)
    grads = ops.qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs, positions)
    for y, g, gw, dy, x, w in ((yq, grads[0], grads[2], dq, q, wq), (yk, grads[1], grads[3], dk, k, wk)):
        want, size = forward(x, w, freqs, positions, 1e-6, False)
        close(y, want, (24 * UNIT + loose) * size)
        dx, bound, dw, dw_bound = backward(dy, x, w, freqs, positions, 1e-6, False)
        close(g, dx, bound * (1 + loose / (48 * UNIT)))
        assert (gw is None) == (w is None)
        if w is not None:
            close(gw, dw, dw_bound * (1 + loose / (48 * UNIT)))


@pytest.mark.parametrize("dtype", TYPES)
def test_any_strides_give_the_same_bits(ops, dtype):
    B, L, hq, hk, d = 2, 21, 3, 2, 32
    q, k, wq, wk, dq, dk, gen = operands(B, L, hq, hk, d, dtype, 4)
    freqs = ops.rope_frequencies(d)
    want = ops.qk_norm_rope(q.contiguous(), k.contiguous(), wq, wk, freqs)
    want_back = ops.qk_norm_rope_backward(dq, dk, q.contiguous(), k.contiguous(), wq, wk, freqs)

    def shifted(t, by):          # the same values from an address that is no multiple of 8 or 16 bytes
        flat = torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")
        flat[by:] = t.reshape(-1)
        return flat[by:].view(t.shape)

    for other in (lambda t: t, lambda t: shifted(t, 1), lambda t: shifted(t, 4), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                  lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)):
        for a, b in zip(ops.qk_norm_rope(other(q), other(k), wq, wk, freqs), want):
            close(a, b.double().cpu(), 24 * UNIT * b.double().cpu().abs().amax(-1, keepdim=True) * 2)
        for a, b in zip(ops.qk_norm_rope_backward(other(dq), other(dk), other(q), other(k), wq, wk, freqs), want_back):
            close(a, b.double().cpu(), 96 * UNIT * 30 * b.double().cpu().abs().amax())
    expanded = q[:1].expand(3, L, hq, d)
    assert torch.equal(ops.qk_norm_rope(expanded, k[:1].expand(3, L, hk, d), wq, wk, freqs)[0][2], want[0][0])


def test_zero_heads_and_what_is_not_finite(ops):
    q = torch.zeros(1, 4, 2, 32, device="cuda")
    q[0, 1, 1, 5] = float("inf")
    q[0, 2, 0, 0] = float("nan")
    w = torch.ones(32, device="cuda")
    freqs = ops.rope_frequencies(32)
    y, _ = ops.qk_norm_rope(q, q, w, w, freqs)
    assert y[0, 0, 2].isnan().all()                                   # (B, h, L, d)
    assert y[0, 1, 1, [5, 21]].isnan().all()                          # infinity times its norm of zero
    keep = torch.ones(2, 4, dtype=torch.bool)
    keep[1, 1] = keep[0, 2] = False
    assert (y[0][keep] == 0).all()
    g = ops.qk_norm_rope_backward(torch.ones_like(y), torch.ones_like(y), torch.zeros_like(q), torch.zeros_like(q), w, w, freqs)
    assert all(t.isfinite().all() for t in g) and (g[2] == 0).all()


def test_gradients_into_a_fused_projection(ops):
    B, L, hq, hk, d = 2, 31, 4, 2, 32
    q, k, wq, wk, dq, dk, gen = operands(B, L, hq, hk, d, torch.float32, 12)
    freqs = ops.rope_frequencies(d)
    want = ops.qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs)
    out = torch.full((B, L, (hq + 2 * hk) * d), 7.0, device="cuda")
    got = ops.qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(out[..., :hq * d], want[0].flatten(2)) and (out[..., (hq + hk) * d:] == 7.0).all()
    with pytest.raises(ValueError):
        ops.qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs, out=q._base)


def test_the_same_gradients_again(ops):
    """The weights' gradients are sums in one order"""
    q, k, wq, wk, dq, dk, _ = operands(4, 500, 8, 4, 32, torch.float32, 1)
    freqs = ops.rope_frequencies(32)
    first = ops.qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(ops.qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs), first))


def test_no_tokens(ops):
    w = torch.ones(8, device="cuda")
    for B, L in ((0, 3), (3, 0)):
        x, g = torch.empty(B, L, 2, 8, device="cuda"), torch.empty(B, 2, L, 8, device="cuda")
        assert ops.qk_norm_rope(x, x, w, w)[0].shape == (B, 2, L, 8)
        gq, gk, gwq, gwk = ops.qk_norm_rope_backward(g, g, x, x, w, w)
        assert gq.shape == (B, L, 2, 8) and (gwq == 0).all() and (gwk == 0).all()


def test_captured_and_replayed(ops):
    q, k, wq, wk, dq, dk, gen = operands(2, 90, 4, 4, 32, torch.float32, 8)
    base, freqs = q._base, ops.rope_frequencies(32)
    positions = torch.arange(90, device="cuda", dtype=torch.int32)

    def both():
        return ops.qk_norm_rope(q, k, wq, wk, freqs, positions) + ops.qk_norm_rope_backward(dq, dk, q, k, wq, wk, freqs, positions)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for _ in range(4):
        base.normal_(generator=gen)
        dq.normal_(generator=gen)
        positions += 17
        graph.replay()
        kept = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(kept, both()))


def test_refusals(ops):
    q, k, wq, wk, dq, dk, _ = operands(2, 3, 2, 1, 8, torch.float32, 2)
    f = ops.rope_frequencies(8)
    for bad in (lambda: ops.qk_norm_rope(q[0], k), lambda: ops.qk_norm_rope(q, k[:, :2]), lambda: ops.qk_norm_rope(q, k[..., :4]),
                lambda: ops.qk_norm_rope(q, k, wq[:4]), lambda: ops.qk_norm_rope(q, k, wq, wk, ops.rope_frequencies(10)),
                lambda: ops.qk_norm_rope(q, k, wq, wk, f, torch.zeros(2, device="cuda", dtype=torch.int32)), lambda: ops.qk_norm_rope(q, k, eps=-1.0),
                lambda: ops.qk_norm_rope(q, k, eps=float("nan")), lambda: ops.qk_norm_rope(q[:, :, :0], k), lambda: ops.rope_frequencies(7),
                lambda: ops.qk_norm_rope(torch.zeros(1, 1, 1, 513, device="cuda"), torch.zeros(1, 1, 1, 513, device="cuda")),
                lambda: ops.qk_norm_rope_backward(dq.transpose(1, 2), dk, q, k), lambda: ops.qk_norm_rope_backward(dq, dq, q, k),
                lambda: ops.qk_norm_rope_backward(dq, dk, q, k, out=torch.zeros(2, 3, 23, device="cuda")),
                lambda: ops.qk_norm_rope_backward(dq, dk, q, k, out=torch.zeros(2, 3, 48, device="cuda")[..., ::2])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.qk_norm_rope(q.double(), k.double()), lambda: ops.qk_norm_rope(q, k.half()), lambda: ops.qk_norm_rope(q.cpu(), k),
                lambda: ops.qk_norm_rope(q, k, wq.half()), lambda: ops.qk_norm_rope(q, k, wq, wk, f.float()),
                lambda: ops.qk_norm_rope(q, k, wq, wk, f, torch.zeros(3, device="cuda")), lambda: ops.qk_norm_rope_backward(dq.half(), dk, q, k),
                lambda: ops.qk_norm_rope_backward(dq, dk, q, k, out=torch.zeros(2, 3, 32, device="cuda").half())):
        with pytest.raises(TypeError):
            bad()


def test_more_heads_than_a_launch_can_number_are_refused(ops):
    q = torch.zeros(1, 1, 1, 4, device="cuda")
    for h in (65536, (1 << 32) + 1):
        for a, b in ((q.expand(1, 1, h, 4), q), (q, q.expand(1, 1, h, 4))):
            with pytest.raises(ValueError):
                ops.qk_norm_rope(a, b)
