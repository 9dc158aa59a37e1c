"""attention.window_attention (csrc/window_attention.hip, window_attention_bwd.hip) against its 64-bit statement, forward and gradients."""
import pytest
import torch

from _attention_ref import close, reference

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _qkv(B, N, M, H, Hk, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((B, N, H, D), (B, M, Hk, D), (B, M, Hk, D), (B, N, H, D))]


def _ints(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")


def _run(q, k, v, do, left, right, sinks, lengths=None, starts=None, scale=None):
    from patchaugnet_amd.attention import window_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = window_attention(*leaves, left=left, right=right, sinks=sinks, scale=scale, lengths=_ints(lengths), q_start=_ints(starts))
    grads = torch.autograd.grad(out, leaves, do)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads))


def _check(q, k, v, do, left, right, sinks, lengths=None, starts=None, scale=None):
    got = _run(q, k, v, do, left, right, sinks, lengths, starts, scale)
    val, tol = reference(q, k, v, left, right, sinks, scale, lengths, starts, do)
    for n in val:
        assert got[n].dtype == q.dtype
        close(got[n], val[n], tol[n], n)
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 72, 96, 128])
def test_head_widths(dtype, D):
    _check(*_qkv(2, 150, 150, 4, 2, D, dtype, seed=D), 37, 0, 3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,left,right,sinks", [
    (1, None, 0, 0), (1, 0, 0, 0), (2, 0, 0, 1), (31, 5, 5, 0), (33, None, None, 0), (64, 63, 0, 0), (65, 64, 0, 64), (127, 0, 0, 0), (129, 0, 127, 2),
    (200, None, 0, 5), (257, 1, 1, 70), (300, 31, 33, 129), (300, 1000, 1000, 7), (513, 128, 0, 300)])
def test_lengths_and_windows(dtype, N, left, right, sinks):
    _check(*_qkv(1, N, N, 2, 1, 32, dtype, seed=N), left, right, sinks)


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 3), (3, 1), (6, 2), (8, 1), (40, 1), (7, 7)])
def test_shared_heads(H, Hk):
    _check(*_qkv(2, 70, 70, H, Hk, 16, F16, seed=H), 20, 0, 4)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_padded_batch(dtype):
    lengths = [130, 0, 1, 64, 77, 200, -3]
    q, k, v, do = _qkv(7, 130, 130, 2, 2, 24, dtype)
    got = _check(q, k, v, do, 17, 9, 2, lengths)
    for b, n in enumerate(lengths):
        n = min(max(n, 0), 130)
        for t in got.values():
            assert not t[b, n:].any()


def test_padding_may_hold_anything():
    """Not a number and infinities in the padding of every input change nothing, in no output."""
    lengths = [100, 3, 0, 65]
    q, k, v, do = _qkv(4, 100, 100, 4, 2, 64, BF16, seed=5)
    clean = _run(q, k, v, do, 30, 5, 2, lengths)
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (do, float("-inf"))):
        for b, n in enumerate(lengths):
            t[b, n:] = bad
    dirty = _run(q, k, v, do, 30, 5, 2, lengths)
    for n in clean:
        assert torch.equal(clean[n], dirty[n]), n


@pytest.mark.parametrize("N,M,starts", [(1, 500, [499, 17]), (5, 300, [0, 295]), (64, 640, [576, 100]), (130, 1000, [870, 3]), (40, 30, [0, 0]), (10, 90, [85, 200])])
def test_parts_of_a_prompt(N, M, starts):
    """Queries behind cached keys; rows past the keys are padding."""
    _check(*_qkv(2, N, M, 4, 1, 32, BF16, seed=M), 90, 0, 4, lengths=[min(M, s + N) for s in starts], starts=starts)


def test_no_keys_and_no_queries():
    from patchaugnet_amd.attention import window_attention
    got = _run(*_qkv(2, 5, 0, 2, 2, 32, F32), None, 0, 0)
    assert not got["out"].any() and not got["dq"].any() and got["dk"].shape == (2, 0, 2, 32)
    got = _run(*_qkv(2, 0, 5, 2, 2, 32, F32), None, 0, 0)
    assert got["out"].shape == (2, 0, 2, 32) and not got["dk"].any() and not got["dv"].any()
    assert window_attention(*_qkv(0, 4, 4, 2, 2, 32, F32)[:3]).shape == (0, 4, 2, 32)


def test_one_visible_key_returns_its_value():
    q, k, v, do = _qkv(1, 200, 200, 2, 2, 64, F16)
    got = _run(q, k, v, do, 0, 0, 0)
    assert torch.equal(got["out"], v) and torch.equal(got["dv"], do)


@pytest.mark.parametrize("amp", [40.0, 300.0])
def test_large_scores(amp):
    """Scores of thousands: one key takes all, the others underflow; nothing overflows."""
    q, k, v, do = _qkv(1, 100, 100, 2, 2, 32, F32, seed=3)
    got = _run(q * amp, k, v, do, 20, 20, 1)
    val, tol = reference(q * amp, k, v, 20, 20, 1, dout=do)
    for n in val:
        close(got[n], val[n], tol[n], n)


def test_growing_scores_rescale():
    """Keys whose scores grow along the sequence move the running maximum in every tile, far beyond the range of one exponent."""
    q, k, v, do = _qkv(1, 400, 400, 1, 1, 32, BF16, seed=4)
    q, k = q.abs(), k.abs() * torch.linspace(0, 30, 400, device="cuda", dtype=BF16).view(1, -1, 1, 1)
    _check(q, k, v, do, None, 0, 0)


def test_views_of_one_projection():
    """q, k, v as views of one (B, N, 3, H, D) tensor, a transposed batch, an expanded gradient; an unaligned view."""
    from patchaugnet_amd.attention import window_attention
    g = torch.Generator(device="cuda").manual_seed(9)
    qkv = torch.randn(2, 90, 3, 4, 32, generator=g, device="cuda").to(BF16)
    q, k, v = qkv.unbind(2)
    do = torch.randn(4, 32, generator=g, device="cuda").to(BF16).expand(2, 90, 4, 32)
    got = _check(q, k, v, do, 16, 0, 1)
    assert torch.equal(got["out"], window_attention(q.contiguous(), k.contiguous(), v.contiguous(), left=16, sinks=1))
    hn = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)                       # heads outside, tokens inside
    assert torch.equal(got["out"], window_attention(hn, k, v, left=16, sinks=1))
    wide = torch.zeros(2, 90, 4, 33, device="cuda", dtype=BF16)
    wide[..., 1:] = q
    assert torch.equal(got["out"], window_attention(wide[..., 1:], k, v, left=16, sinks=1))


def test_same_bits_every_run_and_with_or_without_gradient():
    from patchaugnet_amd.attention import window_attention
    q, k, v, do = _qkv(2, 700, 700, 8, 1, 64, BF16, seed=1)
    a = _run(q, k, v, do, 50, 0, 200)
    for _ in range(3):
        b = _run(q, k, v, do, 50, 0, 200)
        for n in a:
            assert torch.equal(a[n], b[n]), n
    with torch.no_grad():
        assert torch.equal(a["out"], window_attention(q, k, v, left=50, sinks=200))


def test_few_rows_over_many_keys():
    """Few queries over a long sequence: the keys are split over workgroups and joined; gradients of few keys seen by many rows."""
    _check(*_qkv(1, 3, 5000, 4, 4, 64, F16, seed=8), None, 0, 0, lengths=[5000], starts=[4997])
    _check(*_qkv(1, 3000, 3000, 1, 1, 32, F32, seed=8), 40, 0, 5)


def test_gradients_against_differences():
    """Directional differences of the 64-bit forward, step 2^-10: the third derivative's part is below 1e-6 of the sum of |gradient| |direction|."""
    q, k, v, do = _qkv(1, 40, 40, 2, 1, 16, F32, seed=2)
    got = _run(q, k, v, do, 12, 3, 2)
    gen = torch.Generator(device="cuda").manual_seed(77)
    for i, n in enumerate(("dq", "dk", "dv")):
        d = torch.randn((q, k, v)[i].shape, generator=gen, device="cuda").double()
        h = 2.0 ** -10
        f = []
        for sgn in (1, -1):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + sgn * h * d
            out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
            from _attention_ref import seen
            ok = seen(40, 40, 12, 3, 2, 40, 0, "cuda")
            for hd in range(2):
                s = (x[0][0, :, hd] @ x[1][0, :, 0].t().contiguous()) / 4.0
                out[0, :, hd] = torch.softmax(s.masked_fill(~ok, float("-inf")), 1) @ x[2][0, :, 0]
            f.append((out * do.double()).sum())
        diff = (f[0] - f[1]) / (2 * h)
        along = (got[n].double() * d).sum()
        assert abs(float(diff - along)) <= 1e-5 * float((got[n].double() * d).abs().sum()), n


def test_on_another_stream():
    q, k, v, do = _qkv(2, 300, 300, 4, 2, 64, F16, seed=6)
    want = _run(q, k, v, do, 33, 0, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, do, 33, 0, 2)
    side.synchronize()
    for n in want:
        assert torch.equal(want[n], got[n]), n


def test_captured_step_replays():
    """A forward and backward pass captured into a graph, replayed between eager calls with new inputs, equals the eager results."""
    q, k, v, do = _qkv(1, 600, 600, 8, 2, 64, BF16, seed=11)
    lengths = _ints([600])
    from patchaugnet_amd.attention import window_attention
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]

    def step():
        out = window_attention(*leaves, left=70, sinks=4, lengths=lengths)
        return (out.detach(),) + torch.autograd.grad(out, leaves, do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(4):
        fresh = _qkv(1, 600, 600, 8, 2, 64, BF16, seed=20 + turn)
        with torch.no_grad():
            for t, f in zip(leaves, fresh):
                t.copy_(f)
        lengths.fill_(600 - 150 * turn)
        graph.replay()
        torch.cuda.synchronize()
        held_now = [t.clone() for t in held]
        want = _run(*fresh[:3], do, 70, 0, 4, lengths=[600 - 150 * turn])
        for a, b in zip(held_now, want.values()):
            assert torch.equal(a, b), turn


def test_refusals():
    from patchaugnet_amd.attention import window_attention
    q, k, v, _ = _qkv(2, 20, 20, 4, 2, 32, F32)
    for bad, exc in [
            (lambda: window_attention(q.cpu(), k, v), RuntimeError), (lambda: window_attention(q, k.half(), v), TypeError),
            (lambda: window_attention(q.double(), k.double(), v.double()), TypeError), (lambda: window_attention(q[0], k, v), ValueError),
            (lambda: window_attention(q[:, :, :3], k, v), ValueError), (lambda: window_attention(q[..., :12], k[..., :12], v[..., :12]), ValueError),
            (lambda: window_attention(q, k, v[:, :10]), ValueError), (lambda: window_attention(q, k[:1], v[:1]), ValueError),
            (lambda: window_attention(q, k, v, left=-1), ValueError), (lambda: window_attention(q, k, v, right=1.5), ValueError),
            (lambda: window_attention(q, k, v, sinks=-2), ValueError), (lambda: window_attention(q, k, v, scale=0.0), ValueError),
            (lambda: window_attention(q, k, v, scale=float("nan")), ValueError), (lambda: window_attention(q, k, v, lengths=torch.tensor([1, 2])), ValueError),
            (lambda: window_attention(q, k, v, lengths=_ints([1])), ValueError), (lambda: window_attention(q, k, v, q_start=_ints([[1], [2]])), ValueError)]:
        with pytest.raises(exc):
            bad()
    leaf = q.clone().requires_grad_()
    out = window_attention(leaf, k, v)
    (g,) = torch.autograd.grad(out.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (BF16, 96), (F32, 128), (F32, 64)])
@pytest.mark.parametrize("H,Hk", [(4, 1), (3, 1), (2, 2)])
def test_rows_far_behind_the_first_tokens(dtype, D, H, Hk):
    """Many rows that see the first tokens only beyond their window: those gradients are gathered apart and joined.  Two groups of 32 first tokens."""
    _check(*_qkv(1, 900, 900, H, Hk, D, dtype, seed=D + H), 100, 0, 37)
    _check(*_qkv(2, 700, 700, H, Hk, D, dtype, seed=D), 300, 20, 5, lengths=[700, 411])


@pytest.mark.parametrize("H,Hk", [(5, 1), (7, 1), (24, 1), (64, 1), (65, 1), (130, 1)])
def test_large_groups(H, Hk):
    """Groups that do not divide a tile of rows, fill one, and exceed one."""
    _check(*_qkv(1, 60, 60, H, Hk, 32, BF16, seed=H), 11, 4, 2)
    _check(*_qkv(1, 40, 40, H, Hk, 128, F32, seed=H), 11, 0, 1)


def test_keys_behind_four_gigabytes():
    """Keys and values of more than 2^31 elements: the last queries see the last keys and the first ones; all other gradients are zero."""
    M, N, D, left, sinks = 2 ** 24 + 40, 40, 128, 100, 3
    g = torch.Generator(device="cuda").manual_seed(12)
    q, do = (torch.randn(1, N, 2, D, generator=g, device="cuda").to(BF16) for _ in range(2))
    k, v = (torch.zeros(1, M, 1, D, dtype=BF16, device="cuda") for _ in range(2))
    near = torch.cat([torch.arange(sinks), torch.arange(M - N - left - 8, M)]).cuda()
    for t in (k, v):
        t[0, near] = torch.randn(near.numel(), 1, D, generator=g, device="cuda").to(BF16)
    got = _run(q, k, v, do, left, 0, sinks, lengths=[M], starts=[M - N])
    # the same rows over the keys that hold anything: the first ones, then the last ones, which keep their distances to the queries
    ks, vs = k[:, near], v[:, near]
    m = near.numel()
    val, tol = reference(q, ks, vs, left, 0, sinks, None, [m], [m - N], do)
    for n in ("out", "dq"):
        close(got[n], val[n], tol[n], n)
    for n in ("dk", "dv"):
        close(got[n][:, near], val[n], tol[n], n)
        assert int(got[n].count_nonzero()) == int(got[n][:, near].count_nonzero())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("N,H,Hk,D,left,sinks,few", [
    (2, 2, 2, 32, None, 0, True), (3, 4, 1, 64, None, 0, True), (90, 8, 2, 64, 16, 1, True), (300, 4, 4, 128, None, 0, True), (300, 4, 2, 16, 40, 2, True),
    (2100, 4, 2, 64, 511, 4, False), (2100, 4, 2, 128, 511, 4, False), (2100, 4, 2, 16, 511, 4, False)])
def test_error_beside_the_rounding_of_the_result(dtype, N, H, Hk, D, left, sinks, few):
    """2-norm of the error over that of rounding the exact result.  Up to 2^22 pairs products take P and dS in two parts, whose remainder is 2^-8 of a rounding or
    less: even magnified ten times by the difference in dS it adds 1e-3 in the sum of squares.  Above, the rounding of P counts once in out and dv (sqrt 2), that
    of dS once and that of P, through delta, at most once more in dq and dk (sqrt 3): independent errors of the rounding's relative size.  2 % for the sample."""
    assert few == (H * N * min(N, N if left is None else left + 1) <= 1 << 22)
    q, k, v, do = _qkv(1, N, N, H, Hk, D, dtype, seed=11)
    got = _run(q, k, v, do, left, 0, sinks)
    val, _ = reference(q, k, v, left, 0, sinks, None, None, None, do)
    for n, most in (("out", 2), ("dq", 3), ("dk", 3), ("dv", 2)):
        ratio = (got[n].double() - val[n]).norm() / (val[n].to(dtype).double() - val[n]).norm()
        assert ratio <= 1.02 * (1 if few else most) ** 0.5, (n, float(ratio))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_queries_behind_first_tokens(dtype):
    """An empty part of a prompt: nothing sees the keys, their gradients are zeros whatever the window and the first tokens."""
    for left, sinks, starts in ((3, 2, [4, 90]), (0, 40, [0, 0]), (None, 5, [7, 200])):
        got = _run(*_qkv(2, 0, 90, 4, 2, 32, dtype), left, 0, sinks, lengths=[90, 41], starts=starts)
        assert got["out"].shape == got["dq"].shape == (2, 0, 4, 32)
        for n in ("dk", "dv"):
            assert got[n].shape == (2, 90, 2, 32) and not got[n].any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("N,M,lengths,starts,left,right", [
    (100, 100, [65, 3, 0, 100], None, None, 0), (100, 100, [65, 33, 97, 99], None, None, None), (300, 300, [257, 140, 70, 1], None, 200, 40),
    (40, 3000, [3000, 2999, 2961, 5], [2980, 2960, 2960, 0], None, 0)])
def test_padding_beside_rows_that_see_whole_parts(dtype, N, M, lengths, starts, left, right):
    """Padding rows in a wave whose other rows see every key of a 32-key part; the last case splits the keys.  Padding of any value changes nothing, and where
    the sequence itself holds NaN, the padding's output and gradients are still 0."""
    q, k, v, do = _qkv(4, N, M, 4, 2, 64, dtype, seed=5)
    ends = [max(n - (starts[b] if starts else 0), 0) for b, n in enumerate(lengths)]
    clean = _run(q, k, v, do, left, right, 2, lengths, starts)
    for b, n in enumerate(lengths):
        q[b, ends[b]:], do[b, ends[b]:] = float("nan"), float("-inf")
        k[b, n:], v[b, n:] = float("inf"), float("nan")
    dirty = _run(q, k, v, do, left, right, 2, lengths, starts)
    for n in clean:
        assert torch.equal(clean[n], dirty[n]), n
    v[0, 1], k[1, 2], do[2, 0] = float("nan"), float("inf"), float("inf")
    broken = _run(q, k, v, do, left, right, 2, lengths, starts)
    for got in (dirty, broken):
        for b, n in enumerate(lengths):
            assert not got["out"][b, ends[b]:].any() and not got["dq"][b, ends[b]:].any()
            assert not got["dk"][b, n:].any() and not got["dv"][b, n:].any()


def _ratios(got, val, rows=slice(None)):
    """2-norm of the error over that of rounding the exact result, over some rows (or keys)."""
    out = {}
    for n in val:
        g, v = got[n][:, rows].double(), val[n][:, rows]
        out[n] = float((g - v).norm() / (v.to(got[n].dtype).double() - v).norm())
    return out


@pytest.mark.parametrize("N,H,Hk,D,left,sinks,amp", [
    (512, 2, 2, 64, None, 0, 1e-3), (512, 2, 1, 32, 100, 4, 1e-4), (2048, 4, 4, 64, None, 0, 1e-2), (2048, 4, 2, 64, None, 0, 1e-3), (4096, 2, 2, 128, None, 3, 1e-3),
    (16384, 1, 1, 64, None, 0, 1.0), (16384, 1, 1, 64, None, 0, 1e-3), (16384, 1, 1, 16, None, 0, 1.0), (3000, 4, 2, 32, 1023, 40, 1e-3), (3000, 4, 1, 96, 300, 0, 1e-3)])
def test_float16_keeps_digits_of_small_gradients(N, H, Hk, D, left, sinks, amp):
    """Weights of 1 / keys and gradients as a mean loss gives them.  Bounds as in test_error_beside_the_rounding_of_the_result: powers of two that are taken off again
    change no rounding."""
    few = H * N * min(N, N if left is None else left + 1) <= 1 << 22
    q, k, v, do = _qkv(1, N, N, H, Hk, D, F16, seed=11)
    do = do * amp
    got = _run(q, k, v, do, left, 0, sinks)
    val, _ = reference(q, k, v, left, 0, sinks, None, None, None, do)
    for (n, r), most in zip(_ratios(got, val).items(), (2, 3, 3, 2)):
        assert r <= 1.02 * (1 if few else most) ** 0.5, (n, r)


def test_float16_gradients_of_different_sizes():
    """Rows whose gradients are 2^0 .. 2^-11 in turn keep the digits of their own dq; a second half of 2^-13 keeps those of its dk and dv."""
    q, k, v, do = _qkv(1, 2048, 2048, 4, 2, 64, F16, seed=12)
    size = 2.0 ** -(torch.arange(2048, device="cuda") % 12)
    mixed = do * size.to(F16).view(1, -1, 1, 1)
    got = _run(q, k, v, mixed, None, 0, 0)
    val, _ = reference(q, k, v, None, 0, 0, None, None, None, mixed)
    for first in (0, 6, 11):
        r = _ratios({"dq": got["dq"]}, {"dq": val["dq"]}, slice(first, None, 12))["dq"]
        assert r <= 1.02 * 3 ** 0.5, (first, r)
    halves = do * torch.where(torch.arange(2048, device="cuda") < 1024, 1.0, 2.0 ** -13).to(F16).view(1, -1, 1, 1)
    got = _run(q, k, v, halves, 600, 0, 0)
    val, _ = reference(q, k, v, 600, 0, 0, None, None, None, halves)
    for part in (slice(0, 1024), slice(1024 + 128, 2048)):      # keys of the second half are seen by its rows alone
        r = _ratios({n: got[n] for n in ("dk", "dv")}, {n: val[n] for n in ("dk", "dv")}, part)
        assert r["dk"] <= 1.02 * 3 ** 0.5 and r["dv"] <= 1.02 * 2 ** 0.5, (part, r)


@pytest.mark.parametrize("left,sinks", [(3, 0), (None, 2)])
def test_float16_scores_gradients_beyond_its_range(left, sinks):
    """dS of 10^6 and more (large values and gradients) beside keys and queries of 10^-3: the products fit the type, dS alone would not."""
    q, k, v, do = _qkv(1, 200, 200, 4, 2, 32, F16, seed=13)
    do[:, ::7] *= 2.0 ** -12                                    # and rows far below
    _check(q * 2.0 ** -10, k * 2.0 ** -10, v * 64, do * 2.0 ** 13, left, 0, sinks)


def test_strides_of_dimensions_with_one_entry_mean_nothing():
    """One batch, one token, one head: their strides may be anything, a single head cut out of (B, H, N, D) among them."""
    q, k, v, do = _qkv(1, 50, 50, 1, 1, 32, BF16, seed=1)
    want = _run(q, k, v, do, 9, 0, 1)
    odd = [t.as_strided(t.shape, s) for t, s in ((q, (1601, 32, 1 << 23, 1)), (k, (7, 32, 33, 1)), (v, (1, 32, 1 << 30, 1)), (do, (3, 32, 5, 1)))]
    assert all(t.is_contiguous() for t in odd)
    got = _run(*odd, 9, 0, 1)
    for n in want:
        assert torch.equal(want[n], got[n]), n
    one = [t[:, :1] for t in (q, k, v, do)]
    want = _run(*[t.contiguous() for t in one], None, 0, 0)
    got = _run(*[t.as_strided(t.shape, (33, 1 << 23, 17, 1)) for t in one], None, 0, 0)
    for n in want:
        assert torch.equal(want[n], got[n]), n
    N = (1 << 22) // 128 + 5                                    # the head's stride passes 2^22 elements
    q, k, v, do = (torch.randn(1, 1, N, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).to(BF16).transpose(1, 2) for i in range(4))
    got = _run(q, k, v, do, 20, 0, 0)
    want = _run(*[t.squeeze(2).unsqueeze(2).clone(memory_format=torch.contiguous_format) for t in (q, k, v, do)], 20, 0, 0)
    for n in want:
        assert torch.equal(want[n], got[n]), n


def test_more_joined_keys_than_a_launch_holds():
    """2^24 first tokens and some, whose partial sums are joined by a workgroup each: the last ones come out like the first."""
    M = (1 << 24) + 100
    q, k, v, do = _qkv(1, 2, M, 1, 1, 8, BF16, seed=14)
    do = do * 2.0 ** 10
    got = _run(q, k, v, do, 0, None, M, lengths=[M], starts=[0])
    val, _ = reference(q, k, v, 0, None, M, None, [M], [0], do)
    for part in (slice(0, 4096), slice(M - 4096, M)):
        for n in ("dk", "dv"):
            assert val[n][:, part].any()
            assert _ratios({n: got[n]}, {n: val[n]}, part)[n] <= 2.0, (n, part)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("what", ["inf", "nan"])
def test_a_broken_gradient_stays_with_its_keys(dtype, what):
    """An infinity or NaN in one row's incoming gradient: keys in later 32-key parts, which do not see the row, keep their dk and dv, other rows their dq."""
    q, k, v, do = _qkv(1, 1500, 1500, 2, 1, 64, dtype, seed=15)
    do = do * 64
    do[0, 63] = 0
    do[0, 90:] *= 2.0 ** -10                                    # the largest dS that keys from 64 on meet stand beside the broken row, or just behind
    v[0, :32, 0, 7], v[0, 32:64, 0, 7] = 9, -0.5                # the gradients of the row's weights: NaN in its first part, minus infinity in its second
    val, _ = reference(q, k, v, None, 0, 0, None, None, None, do)
    do[0, 63, 1, 7] = float(what)
    got = _run(q, k, v, do, None, 0, 0)
    late = slice(64, None)
    for n in ("dq", "dk", "dv"):
        assert torch.isfinite(got[n][:, late]).all(), n
        assert (got[n][:, late].double() - val[n][:, late]).norm() <= 4 * (torch.finfo(dtype).eps / 2 if dtype != F32 else 1e-6) * val[n][:, late].norm(), n
    assert not torch.isfinite(got["dq"][0, 63, 1]).all()
