"""attention.qk_norm_rotary (csrc/qk_norm_rotary.hip) against its 64-bit statement, forward and gradients.

Bounds, to first order, with w = 2^-24 and u half a step of the type: the mean square of D terms and its root, the products and the rotation are off by
w (D + 16) relative; an angle by 2^-25 of its eighth turn, w absolute; so an output by u |y| + w (D + 20) (|n_u| + |n_v|) over its pair.  Gradients likewise
with the sums of their terms' magnitudes; weight gradients are 32-bit sums of B N heads terms."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
W = 2.0 ** -24


def _rotate(x, cos, sin, inter, mag=False):
    """x (B, N, H, D); cos, sin (B, N, P) or None.  mag: sums of magnitudes in place of differences."""
    if cos is None:
        return x
    P = cos.shape[-1]
    c, s = cos.unsqueeze(2), sin.unsqueeze(2)
    iu, iv = (torch.arange(P) * 2, torch.arange(P) * 2 + 1) if inter else (torch.arange(P), torch.arange(P) + P)
    y = x.clone()
    u, v = x[..., iu], x[..., iv]
    if mag:
        y[..., iu] = u + v
        y[..., iv] = u + v
    else:
        y[..., iu], y[..., iv] = u * c - v * s, u * s + v * c
    return y


def _reference(x, w, cos, sin, eps, inter, dy=None):
    u = torch.finfo(x.dtype).eps / 2
    D = x.shape[-1]
    X = x.double()
    r = (X.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = X * r
    wd = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    y = _rotate(n * wd, cos, sin, inter)
    tiny = torch.finfo(x.dtype).smallest_normal * u * 2
    out = {"y": (y, u * y.abs() + W * (D + 20) * _rotate((n * wd).abs(), cos, sin, inter, True) + tiny)}
    if dy is None:
        return out
    s = _rotate(dy.double(), cos, None if sin is None else -sin, inter)
    sa = _rotate(dy.double().abs(), cos, sin, inter, True)
    t, ta = s * wd, sa * wd.abs()
    m, ma = (t * n).mean(-1, keepdim=True), (ta * n.abs()).mean(-1, keepdim=True)
    dx = r * (t - n * m)
    out["dx"] = dx, u * dx.abs() + W * (3 * D + 60) * r * (ta + n.abs() * ma) + tiny
    terms = dy.shape[0] * dy.shape[1] * dy.shape[2]
    dw = (s * n).sum((0, 1, 2))
    uw = u if w is not None and w.dtype != F32 else 0.0
    out["dw"] = dw, uw * dw.abs() + W * (terms + D + 40) * (sa * n.abs()).sum((0, 1, 2)) + tiny
    return out


def _close(got, want, what):
    val, tol = want
    err = (got.double() - val).abs()
    assert not (~(err <= tol)).any(), (what, float((err / tol).max()))


def _angles(pos, freq, B, N):
    """pos (N,), (B, N), (N, A) or (B, N, A); freq (A, F)"""
    A = freq.shape[0]
    p = pos.double()
    if A == 1 and p.shape in ((N,), (B, N)):
        p = p.unsqueeze(-1)
    p = p.expand(B, N, A)
    a = (p.unsqueeze(-1) * freq.double()).flatten(2)
    return a.cos(), a.sin()


def _check(B, N, H, Hk, D, dtype, freq=None, pos=None, inter=False, wdtype=F32, seed=0, eps=1e-6, scale=1.0):
    from patchaugnet_amd.attention import qk_norm_rotary
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, gq, gk = (scale * torch.randn(B, N, h, D, generator=g, device="cuda") for h in (H, Hk, H, Hk))
    q, k, gq, gk = (t.to(dtype) for t in (q, k, gq, gk))
    qw, kw = ((None, None) if wdtype is None else ((1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(wdtype) for _ in range(2)))
    leaves = [t.requires_grad_() for t in (q, k, qw, kw) if t is not None]
    out = qk_norm_rotary(q, k, qw, kw, positions=pos, inv_freq=freq, eps=eps, interleaved=inter)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    cos, sin = (None, None) if freq is None else _angles(pos, freq if freq.dim() == 2 else freq.view(1, -1), B, N)
    for i, (x, w, dy) in enumerate(((q, qw, gq), (k, kw, gk))):
        want = _reference(x.detach(), None if w is None else w.detach(), cos, sin, eps, inter, dy)
        assert out[i].dtype == dtype and out[i].is_contiguous()
        _close(out[i].detach(), want["y"], ("y", i))
        _close(grads[i], want["dx"], ("dx", i))
        if w is not None:
            assert grads[2 + i].dtype == w.dtype
            _close(grads[2 + i], want["dw"], ("dw", i))
    return q.detach(), k.detach(), out


def _freq(A, F):
    return (3.0 * 0.8 ** torch.arange(A * F, device="cuda", dtype=torch.float32)).view(A, F)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,P", [(1, 0), (2, 1), (7, 3), (8, 2), (16, 8), (30, 9), (40, 20), (64, 32), (64, 30), (66, 33), (80, 24), (96, 48), (128, 64), (128, 60),
                                 (130, 64), (256, 128), (510, 255), (511, 100), (512, 256)])
@pytest.mark.parametrize("inter", [False, True])
def test_widths(dtype, D, P, inter):
    _check(2, 9, 3, 2, D, dtype, freq=_freq(1, P) if P else None, pos=torch.arange(9, device="cuda", dtype=torch.int32) if P else None, inter=inter, seed=D)


@pytest.mark.parametrize("B,N,H,Hk", [(1, 1, 1, 1), (1, 1, 64, 8), (3, 17, 5, 1), (2, 1000, 4, 4), (40, 33, 8, 2), (1, 5000, 2, 1), (1, 3, 300, 1)])
def test_token_and_head_counts(B, N, H, Hk):
    _check(B, N, H, Hk, 32, BF16, freq=_freq(1, 16), pos=torch.arange(N, device="cuda"), seed=N)


@pytest.mark.parametrize("kind", ["float32", "own type", "none"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weights(kind, dtype):
    _check(2, 50, 2, 2, 64, dtype, wdtype={"float32": F32, "own type": dtype, "none": None}[kind], seed=3)


@pytest.mark.parametrize("A,F", [(1, 10), (2, 8), (3, 10), (3, 1)])
@pytest.mark.parametrize("shared", [False, True])
def test_coordinates(A, F, shared):
    g = torch.Generator(device="cuda").manual_seed(A)
    pos = 2 * torch.rand(*((70,) if shared else (3, 70)), A, generator=g, device="cuda") - 1
    _check(3, 70, 4, 4, 64, F32, freq=_freq(A, F) * 60, pos=pos, seed=A)


def test_far_positions():
    """Angles of positions up to 10^8, and coordinates of 10^5, keep 32-bit accuracy."""
    pos = torch.tensor([0, 1, 10 ** 6, 10 ** 8 + 1, -(10 ** 7)], device="cuda", dtype=torch.int64)
    _check(1, 5, 2, 1, 64, F32, freq=_freq(1, 32), pos=pos)
    _check(1, 5, 2, 1, 64, F32, freq=_freq(1, 32), pos=torch.tensor([1e5, -3.25e4, 0.5, 7.0, -0.0], device="cuda"))


def test_position_zero_is_the_norm_alone():
    q, k, _ = _check(1, 4, 2, 2, 64, F16)
    from patchaugnet_amd.attention import qk_norm_rotary
    a = qk_norm_rotary(q, k)
    b = qk_norm_rotary(q, k, positions=torch.zeros(4, dtype=torch.int32, device="cuda"), inv_freq=_freq(1, 32))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("scale", [1e-4, 1.0, 100.0])
def test_magnitudes(scale):
    _check(2, 20, 2, 1, 48, F32, freq=_freq(1, 8), pos=torch.arange(20, device="cuda"), scale=scale, seed=5)


def test_zero_rows():
    from patchaugnet_amd.attention import qk_norm_rotary
    q = torch.zeros(1, 3, 2, 32, device="cuda", requires_grad=True)
    out = qk_norm_rotary(q, q.detach())
    (g,) = torch.autograd.grad(out[0], q, torch.ones_like(q))
    assert not out[0].any() and torch.isfinite(g).all()


def test_views():
    """Heads of one projection, tokens transposed, an odd offset, an expanded gradient."""
    from patchaugnet_amd.attention import qk_norm_rotary
    g = torch.Generator(device="cuda").manual_seed(1)
    pos, fr = torch.arange(30, device="cuda"), _freq(1, 32)
    qkv = torch.randn(2, 30, 8, 64, generator=g, device="cuda").to(BF16)
    q, k = qkv[:, :, :4], qkv[:, :, 4:6]
    want = qk_norm_rotary(q.contiguous(), k.contiguous(), positions=pos, inv_freq=fr)
    odd = torch.zeros(2, 30, 4, 65, dtype=BF16, device="cuda")
    odd[..., 1:] = q
    for qq in (q, q.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3), q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), odd[..., 1:]):
        leaf = qq.detach().requires_grad_()
        got = qk_norm_rotary(leaf, k, positions=pos, inv_freq=fr)
        assert (got[0].double() - want[0].double()).abs().max() <= 2.0 ** -8 * want[0].double().abs().max() and torch.equal(got[1], want[1])
        dy = torch.randn(64, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(BF16).expand(2, 30, 4, 64)
        (gr,) = torch.autograd.grad(got[0], leaf, dy)
        a = fr.view(1, -1).double()
        cos, sin = _angles(pos, a, 2, 30)
        _close(gr, _reference(q, None, cos, sin, 1e-6, False, dy)["dx"], "dx")


def test_empty_batch():
    from patchaugnet_amd.attention import qk_norm_rotary
    q = torch.zeros(0, 5, 2, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    out = qk_norm_rotary(q, q.detach(), w)
    g = torch.autograd.grad(out[0].sum(), (q, w))
    assert g[0].shape == q.shape and not g[1].any()


def test_gradients_against_differences():
    """Directional differences of the 64-bit forward with step 2^-12: what the third derivative adds is below 1e-6 of the sum of magnitudes."""
    from patchaugnet_amd.attention import qk_norm_rotary
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(1, 6, 2, 24, generator=g, device="cuda").requires_grad_()
    w = (1 + 0.1 * torch.randn(24, generator=g, device="cuda")).requires_grad_()
    pos, fr = torch.arange(6, device="cuda"), _freq(1, 8)
    dy = torch.randn(1, 6, 2, 24, generator=g, device="cuda")
    grads = torch.autograd.grad(qk_norm_rotary(q, q.detach(), w, positions=pos, inv_freq=fr)[0], (q, w), dy)
    cos, sin = _angles(pos, fr, 1, 6)

    def f(x, ww):
        return (_rotate(x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * ww, cos, sin, False) * dy.double()).sum()

    h = 2.0 ** -12
    for i in range(2):
        d = torch.randn((q, w)[i].shape, generator=g, device="cuda").double()
        x = [[t.detach().double() for t in (q, w)] for _ in range(2)]
        x[0][i] = x[0][i] + h * d
        x[1][i] = x[1][i] - h * d
        diff = (f(*x[0]) - f(*x[1])) / (2 * h)
        along = (grads[i].double() * d).sum()
        assert abs(float(diff - along)) <= 1e-5 * float((grads[i].double() * d).abs().sum())


def test_same_bits_and_captured_step():
    from patchaugnet_amd.attention import qk_norm_rotary
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k = (torch.randn(2, 700, h, 64, generator=g, device="cuda").to(F16).requires_grad_() for h in (6, 2))
    w = torch.ones(64, device="cuda", requires_grad=True)
    pos, fr = torch.arange(700, device="cuda"), _freq(1, 32)
    dy = torch.randn_like(q), torch.randn_like(k)

    def step():
        out = qk_norm_rotary(q, k, w, w, positions=pos, inv_freq=fr)
        return tuple(o.detach() for o in out) + torch.autograd.grad(out, (q, k, w), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(3):
        with torch.no_grad():
            q.normal_()
            k.normal_()
            pos.add_(1000)
        graph.replay()
        torch.cuda.synchronize()
        now = [t.clone() for t in held]
        for a, b in zip(now, step()):
            assert torch.equal(a, b), turn


def test_refusals():
    from patchaugnet_amd.attention import qk_norm_rotary
    q, k = torch.zeros(2, 5, 4, 32, device="cuda"), torch.zeros(2, 5, 2, 32, device="cuda")
    w, pos, fr = torch.ones(32, device="cuda"), torch.arange(5, device="cuda"), _freq(1, 16)
    for bad, exc in [
            (lambda: qk_norm_rotary(q.cpu(), k), RuntimeError), (lambda: qk_norm_rotary(q, k.half()), TypeError), (lambda: qk_norm_rotary(q, k[:, :4]), ValueError),
            (lambda: qk_norm_rotary(q, k[..., :8]), ValueError), (lambda: qk_norm_rotary(q[0], k[0]), ValueError), (lambda: qk_norm_rotary(q, k, w[:8]), ValueError),
            (lambda: qk_norm_rotary(q, k, w.half()), ValueError), (lambda: qk_norm_rotary(q.half(), k.half(), w, w.half()), ValueError),
            (lambda: qk_norm_rotary(q, k, w.cpu()), ValueError), (lambda: qk_norm_rotary(q, k, eps=-1.0), ValueError),
            (lambda: qk_norm_rotary(q, k, positions=pos), ValueError), (lambda: qk_norm_rotary(q, k, inv_freq=fr), ValueError),
            (lambda: qk_norm_rotary(q, k, positions=pos, inv_freq=_freq(1, 17)), ValueError),
            (lambda: qk_norm_rotary(q, k, positions=pos[:4], inv_freq=fr), ValueError), (lambda: qk_norm_rotary(q, k, positions=pos, inv_freq=_freq(3, 2)), ValueError),
            (lambda: qk_norm_rotary(q, k, positions=pos.double(), inv_freq=fr), TypeError), (lambda: qk_norm_rotary(q, k, positions=pos, inv_freq=fr.double()), ValueError),
            (lambda: qk_norm_rotary(q, k, positions=pos, inv_freq=fr.clone().requires_grad_()), RuntimeError),
            (lambda: qk_norm_rotary(torch.zeros(1, 1, 1, 513, device="cuda"), torch.zeros(1, 1, 1, 513, device="cuda")), ValueError)]:
        with pytest.raises(exc):
            bad()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,P", [(16, 1), (16, 3), (32, 15), (48, 21), (64, 31), (96, 17), (128, 21), (128, 63), (192, 95), (256, 5), (512, 255), (66, 32), (132, 33)])
@pytest.mark.parametrize("inter", [False, True])
def test_pair_counts_that_leave_half_a_piece(dtype, D, P, inter):
    """Pairs whose second halves, or whose rest, do not start at a whole piece: exchanged between lanes.  More rows than one turn holds."""
    pos = torch.arange(150, device="cuda", dtype=torch.int32)
    _check(1, 150, 3, 1, D, dtype, freq=_freq(1, P), pos=pos, inter=inter, seed=D + P)


def test_positions_of_one_token():
    """(N,), (B, N), (N, 1) and (B, N, 1) name the same positions where they can be mistaken for each other."""
    from patchaugnet_amd.attention import qk_norm_rotary
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k = (torch.randn(2, 1, 2, 16, generator=g, device="cuda") for _ in range(2))
    fr = _freq(1, 8)
    want = qk_norm_rotary(q, k, positions=torch.tensor([[5], [5]], device="cuda"), inv_freq=fr)
    for pos in (torch.tensor([5], device="cuda"), torch.tensor([[5]], device="cuda"), torch.tensor([[[5]], [[5]]], device="cuda")):
        got = qk_norm_rotary(q, k, positions=pos, inv_freq=fr.view(-1) if pos.dim() == 1 else fr)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,P", [(260, 129), (300, 149), (300, 3), (508, 253), (508, 127)])
@pytest.mark.parametrize("inter", [False, True])
def test_exchanged_pairs_of_wide_heads(dtype, D, P, inter):
    """Rows of more than 64 pieces, two to a lane: a pair's halves lie in different pieces of the lanes."""
    _check(1, 150, 3, 1, D, dtype, freq=_freq(1, P), pos=torch.arange(150, device="cuda", dtype=torch.int32), inter=inter, seed=D + P)


@pytest.mark.parametrize("dtype,shift", [(F32, 2), (F16, 2), (BF16, 2), (F32, 1), (BF16, 1)])
@pytest.mark.parametrize("P", [255, 201, 66])
def test_offset_views_of_wide_heads(dtype, shift, P):
    """Rows of 512 that start at 8 or 4 bytes (float32), 4 or 2 bytes (16-bit): narrower pieces, up to four to a lane."""
    from patchaugnet_amd.attention import qk_norm_rotary
    g = torch.Generator(device="cuda").manual_seed(P)
    wide, dy = (torch.randn(2, 40, 3, w, generator=g, device="cuda").to(dtype) for w in (512 + shift, 512))
    q = wide[..., shift:].detach().requires_grad_()
    pos, fr = torch.arange(40, device="cuda"), _freq(1, P)
    out = qk_norm_rotary(q, q.detach(), positions=pos, inv_freq=fr)
    (dq,) = torch.autograd.grad(out[0], q, dy)
    want = _reference(q.detach(), None, *_angles(pos, fr, 2, 40), 1e-6, False, dy)
    for got, n in ((out[0].detach(), "y"), (out[1], "y"), (dq, "dx")):
        _close(got, want[n], n)


def test_more_turns_than_workgroups():
    """2^26 tokens and some: the forward pass's workgroups take further turns; every token as in calls of 2^24."""
    from patchaugnet_amd.attention import qk_norm_rotary
    N = (1 << 26) + 100
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(1, N, 1, 8, generator=g, device="cuda", dtype=BF16)
    pos, fr = torch.arange(N, device="cuda", dtype=torch.int32), _freq(1, 4)
    whole = qk_norm_rotary(q, q[:, :N], positions=pos, inv_freq=fr)
    for i in range(0, N, 1 << 24):
        part = qk_norm_rotary(q[:, i:i + (1 << 24)], q[:, i:i + (1 << 24)], positions=pos[i:i + (1 << 24)], inv_freq=fr)
        assert torch.equal(part[0], whole[0][:, i:i + (1 << 24)]) and torch.equal(part[1], whole[1][:, i:i + (1 << 24)]), i


@pytest.mark.parametrize("dtype,scale,eps", [(F32, 1e25, 1e-6), (BF16, 1e25, 1e-6), (F32, 3e37, 1e-6), (BF16, 1e19, 0.0), (F32, 1e-25, 0.0), (BF16, 1e-30, 0.0),
                                             (F32, 1e-18, 1e-36), (F32, 1e-30, 1e-38)])
def test_rows_whose_squares_leave_32_bits(dtype, scale, eps):
    """Rows of 10^19 and more, and small ones under a small eps: the mean square is neither infinite nor 0.  Gradients of rows that large are below 32 bits' range."""
    q, k = (torch.randn(2, 9, h, 48, generator=torch.Generator(device="cuda").manual_seed(h), device="cuda").mul(scale).to(dtype) for h in (3, 2))
    from patchaugnet_amd.attention import qk_norm_rotary
    pos, fr = torch.arange(9, device="cuda"), _freq(1, 8)
    leaf, gy = q.clone().requires_grad_(), torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda").to(dtype)
    out = qk_norm_rotary(leaf, k, positions=pos, inv_freq=fr, eps=eps)
    (dq,) = torch.autograd.grad(out[0], leaf, gy)
    want = _reference(q, None, *_angles(pos, fr, 2, 9), eps, False, gy)
    _close(out[0].detach(), want["y"], "y")
    _close(out[1], _reference(k, None, *_angles(pos, fr, 2, 9), eps, False)["y"], "k")
    _close(dq, want["dx"], "dx")
    mixed = q.clone()
    mixed[0, 0, 0, 5], mixed[1, 2, 1, 3] = float("inf"), float("nan")
    got = qk_norm_rotary(mixed, k, positions=pos, inv_freq=fr, eps=eps)[0]
    other = torch.ones(q.shape[:3], dtype=torch.bool, device="cuda")
    other[0, 0, 0] = other[1, 2, 1] = False
    assert torch.equal(got[other], out[0].detach()[other]) and got[1, 2, 1].isnan().all()
