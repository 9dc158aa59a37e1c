"""attention.paged_append and attention.paged_attention (csrc/paged_attention.hip) against the 64-bit statement of the windowed attention, and the
serving sequence norm + rotation -> prompt -> append -> one token at a time."""
import pytest
import torch

from _attention_ref import close, reference

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _i(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache(k, v, page, lengths, seed=0, spare=2, order=None):
    """k, v (B, M, Hk, D) dealt out to pages in a random order; rows of no sequence hold NaN."""
    B, M, Hk, D = k.shape
    per = [-(-n // page) for n in lengths]
    total = sum(per) + spare
    ids = torch.randperm(total, generator=torch.Generator().manual_seed(seed))
    kp, vp = (torch.full((total, page, Hk, D), float("nan"), dtype=k.dtype, device="cuda") for _ in range(2))
    table = torch.full((B, max(max(per), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        for e in range(per[b]):
            p = int(ids[at])
            at += 1
            table[b, e] = p
            m = min(page, n - e * page)
            kp[p, :m] = k[b, e * page:e * page + m]
            vp[p, :m] = v[b, e * page:e * page + m]
    return kp, vp, table.cuda()


def _inputs(B, M, H, Hk, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((B, H, D), (B, M, Hk, D), (B, M, Hk, D))]


def _want(q, k, v, lengths, left, sinks, scale=None):
    val, tol = reference(q.unsqueeze(1), k, v, left, 0, sinks, scale, lengths, [max(n - 1, 0) for n in lengths])
    return val["out"][:, 0], tol["out"][:, 0]


def _check(B, lengths, H, Hk, D, dtype, page, left, sinks, seed=0, scale=None):
    from patchaugnet_amd.attention import paged_attention
    q, k, v = _inputs(B, max(max(lengths), 1), H, Hk, D, dtype, seed)
    kp, vp, table = _cache(k, v, page, lengths, seed)
    got = paged_attention(q, kp, vp, table, _i(lengths), left=left, sinks=sinks, scale=scale)
    assert got.dtype == dtype
    close(got, *_want(q, k, v, lengths, left, sinks, scale), "out")
    return q, kp, vp, table, got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 80, 96, 128])
def test_head_widths(dtype, D):
    _check(3, [70, 1, 133], 4, 2, D, dtype, 16, None, 0, seed=D)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 32, 100, 1000])
@pytest.mark.parametrize("left,sinks", [(None, 0), (0, 0), (40, 4), (31, 33), (500, 1)])
def test_pages_and_windows(page, left, sinks):
    _check(4, [0, 5, 64, 333], 2, 2, 32, F16, page, left, sinks, seed=page)


@pytest.mark.parametrize("H,Hk", [(1, 1), (8, 1), (6, 3), (32, 1), (33, 1), (80, 2)])
def test_shared_heads(H, Hk):
    _check(2, [50, 200], H, Hk, 64, BF16, 16, None, 0, seed=H)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths,left,sinks", [([4000, 17, 2500, 0], None, 0), ([9000], None, 0), ([6000, 600], 3000, 40), ([513, 512, 511], None, 0)])
def test_long_caches_split_and_join(dtype, lengths, left, sinks):
    _check(len(lengths), lengths, 4, 2, 64, dtype, 64, left, sinks, seed=1, scale=0.2)


def test_pages_given_back_are_not_read():
    """Entries behind the window may be -1 or any number outside the pool; inside the view such a page holds no keys."""
    from patchaugnet_amd.attention import paged_attention
    q, kp, vp, table, got = _check(2, [900, 700], 4, 2, 32, BF16, 16, 100, 3, seed=3)
    holes = table.clone()
    holes[0, 1:(899 - 100) // 16] = -1
    holes[1, 1:(699 - 100) // 16] = 2 ** 31 - 1
    assert torch.equal(got, paged_attention(q, kp, vp, holes, _i([900, 700]), left=100, sinks=3))
    # all pages gone but the last: 900 = 56 * 16 + 4 keys
    holes[0, :-1] = -5
    alone = paged_attention(q, kp, vp, holes, _i([900, 700]), left=100, sinks=3)[0]
    last = paged_attention(q[:1], kp, vp, table[:1, 56:].contiguous(), _i([4]))[0]
    eps = torch.finfo(BF16).eps
    assert (alone.double() - last.double()).abs().max() <= 2 * eps * last.double().abs().max()
    holes.fill_(-1)
    assert not paged_attention(q, kp, vp, holes, _i([900, 700]), left=100, sinks=3).any()


def test_lengths_outside_the_table_are_clamped():
    from patchaugnet_amd.attention import paged_attention
    q, kp, vp, table, got = _check(2, [64, 48], 2, 2, 32, F32, 16, None, 0)
    assert torch.equal(got[:1], paged_attention(q[:1], kp, vp, table[:1], _i([10 ** 6])))
    assert not paged_attention(q, kp, vp, table, _i([-7, 0])).any()
    empty = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    assert not paged_attention(q, kp, vp, empty, _i([5, 5])).any()
    assert not paged_attention(q, kp[:0], vp[:0], table, _i([64, 48])).any()
    assert paged_attention(q[:0], kp, vp, table[:0], _i([])).shape == (0, 2, 32)


def test_pool_layouts():
    """Keys and values side by side in one pool, and pages with the heads outside."""
    from patchaugnet_amd.attention import paged_attention
    q, kp, vp, table, got = _check(2, [64, 48], 4, 2, 32, BF16, 16, None, 0)
    both = torch.stack([kp, vp], 1)
    assert torch.equal(got, paged_attention(q, both[:, 0], both[:, 1], table, _i([64, 48])))
    outside = kp.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(got, paged_attention(q, outside, vp, table, _i([64, 48])))
    wide = torch.zeros(2, 4, 64, dtype=BF16, device="cuda")
    wide[..., 1::2] = q
    assert torch.equal(got, paged_attention(wide[..., 1::2], kp, vp, table, _i([64, 48])))


def test_rows_behind_four_gigabytes():
    """A pool whose far pages lie beyond 2^31 elements and 2^32 bytes."""
    from patchaugnet_amd.attention import paged_append, paged_attention
    q, k, v = _inputs(1, 40, 2, 2, 64, F16, seed=5)
    page = 32
    pages = (2 ** 31) // (page * 2 * 64) + 8
    pool = torch.zeros(pages, page, 2, 64, dtype=F16, device="cuda")
    table = _i([[pages - 1, pages - 3]])
    vpool = torch.zeros(pages, page, 2, 64, dtype=F16, device="cuda")
    paged_append(k, v, pool, vpool, table, _i([0]))
    assert torch.equal(pool[pages - 1], k[0, :32]) and torch.equal(vpool[pages - 3, :8], v[0, 32:])
    assert int(pool.count_nonzero()) == int(k.count_nonzero())
    close(paged_attention(q, pool, vpool, table, _i([40])), *_want(q, k, v, [40], None, 0), "out")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("T,page,D", [(1, 16, 64), (7, 3, 8), (50, 16, 40), (33, 64, 128)])
def test_append(dtype, T, page, D):
    from patchaugnet_amd.attention import paged_append
    g = torch.Generator(device="cuda").manual_seed(T)
    B, Hk, width = 4, 3, 6
    k, v = (torch.randn(B, T, Hk, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    kp, vp = (torch.randn(40, page, Hk, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    table = torch.randperm(40, generator=torch.Generator().manual_seed(T))[:B * width].view(B, width).to(torch.int32)
    table[1, 2], table[2, 0] = -1, 40
    starts, counts = [0, page - 1, 2, width * page - 2], [T, T + 5, 0, T]
    kw, vw = kp.clone(), vp.clone()
    for b in range(B):
        for t in range(min(T, counts[b])):
            j = starts[b] + t
            if j < width * page and 0 <= int(table[b, j // page]) < 40:
                kw[int(table[b, j // page]), j % page] = k[b, t]
                vw[int(table[b, j // page]), j % page] = v[b, t]
    paged_append(k, v, kp, vp, table.cuda(), _i(starts), counts=_i(counts))
    assert torch.equal(kp, kw) and torch.equal(vp, vw)
    before = kp.clone()
    paged_append(k, v, kp, vp, table.cuda(), _i([-T, 10 ** 9, 2 ** 31 - 1, -2 ** 31]))          # positions outside the table
    assert torch.equal(kp, before)


def test_served_stream_equals_the_prompt():
    """Norm + rotation, a prompt of 37 tokens through window_attention and into the cache, then tokens one at a time: each step equals the row that
    window_attention gives for the whole sequence, to the roundings of the weights (16-bit P, both sides) and of the output."""
    from patchaugnet_amd.attention import paged_append, paged_attention, qk_norm_rotary, window_attention
    B, N, H, Hk, D, page, left, sinks = 2, 60, 4, 2, 64, 16, 20, 2
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(B, N, h, D, generator=g, device="cuda").to(BF16) for h in (H, Hk, Hk))
    w = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    freq = 10000.0 ** (-torch.arange(D // 2, device="cuda") / (D // 2))
    pos = torch.arange(N, device="cuda", dtype=torch.int32)
    qr, kr = qk_norm_rotary(q, k, w, w, positions=pos, inv_freq=freq)
    whole = window_attention(qr, kr, v, left=left, sinks=sinks)
    val, tol = reference(qr, kr, v, left, 0, sinks)
    close(whole, val["out"], tol["out"], "prompt")

    width = -(-N // page)
    kp, vp = (torch.full((B * width, page, Hk, D), float("nan"), dtype=BF16, device="cuda") for _ in range(2))
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(1)).view(B, width).to(torch.int32).cuda()
    start = 37
    qp, kk = qk_norm_rotary(q[:, :start], k[:, :start], w, w, positions=pos[:start], inv_freq=freq)
    assert torch.equal(kk, kr[:, :start])
    paged_append(kk, v[:, :start], kp, vp, table, _i([0, 0]))
    for t in range(start, N):
        q1, k1 = qk_norm_rotary(q[:, t:t + 1], k[:, t:t + 1], w, w, positions=pos[t:t + 1], inv_freq=freq)
        paged_append(k1, v[:, t:t + 1], kp, vp, table, _i([t, t]))
        out = paged_attention(q1[:, 0], kp, vp, table, _i([t + 1, t + 1]), left=left, sinks=sinks)
        close(out, val["out"][:, t], tol["out"][:, t], t)


def test_captured_step_replays():
    """One serving step (append and attention, split and joined) captured; lengths, table and inputs change between replays."""
    from patchaugnet_amd.attention import paged_append, paged_attention
    B, M, H, Hk, D, page = 2, 3000, 4, 2, 64, 64
    q, k, v = _inputs(B, M, H, Hk, D, BF16, seed=7)
    kp, vp, table = _cache(k, v, page, [M, M])
    k1, v1 = k[:, -1:].clone(), v[:, -1:].clone()
    lengths, starts = _i([100, 2000]), _i([99, 1999])

    def step():
        paged_append(k1, v1, kp, vp, table, starts)
        return paged_attention(q, kp, vp, table, lengths)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in ([100, 2000], [3000, 1], [1, 2999], [640, 641]):
        q.normal_()
        k1.normal_()
        lengths.copy_(_i(n))
        starts.copy_(_i([i - 1 for i in n]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, paged_attention(q, kp, vp, table, lengths)), n


def test_refusals():
    from patchaugnet_amd.attention import paged_append, paged_attention
    q, k, v = _inputs(2, 16, 4, 2, 32, BF16)
    kp, vp, table = _cache(k, v, 16, [16, 16])
    ln = _i([16, 16])
    skew = torch.zeros(4, 16, 2, 33, dtype=BF16, device="cuda")[..., 1:]
    for bad, exc in [
            (lambda: paged_attention(q.cpu(), kp, vp, table, ln), RuntimeError), (lambda: paged_attention(q.float(), kp, vp, table, ln), TypeError),
            (lambda: paged_attention(q.unsqueeze(1), kp, vp, table, ln), ValueError), (lambda: paged_attention(q[:, :3], kp, vp, table, ln), ValueError),
            (lambda: paged_attention(q, kp, vp[:1], table, ln), ValueError), (lambda: paged_attention(q, kp, vp, table.long(), ln), ValueError),
            (lambda: paged_attention(q, kp, vp, table[:1], ln), ValueError), (lambda: paged_attention(q, kp, vp, table, ln[:1]), ValueError),
            (lambda: paged_attention(q, kp, vp, table, None), ValueError), (lambda: paged_attention(q, kp, vp, table, ln, left=-3), ValueError),
            (lambda: paged_attention(q, skew, skew, table, ln), ValueError), (lambda: paged_attention(q, kp[:, :0], vp[:, :0], table, ln), ValueError),
            (lambda: paged_attention(q.clone().requires_grad_(), kp, vp, table, ln), RuntimeError),
            (lambda: paged_attention(q, kp, vp, table, ln, scale=-1.0), ValueError),
            (lambda: paged_append(k, v[:, :3], kp, vp, table, ln), ValueError), (lambda: paged_append(k[:, :, :1], v[:, :, :1], kp, vp, table, ln), ValueError),
            (lambda: paged_append(k, v, kp, vp, table, None), ValueError), (lambda: paged_append(k, v, kp, vp, table, ln.float()), ValueError),
            (lambda: paged_append(k.float(), v.float(), kp, vp, table, ln), TypeError), (lambda: paged_append(k, v, skew, skew, table, ln), ValueError),
            (lambda: paged_append(k.clone().requires_grad_(), v, kp, vp, table, ln), RuntimeError)]:
        with pytest.raises(exc):
            bad()
    with torch.no_grad():
        paged_attention(q.clone().requires_grad_(), kp, vp, table, ln)


def test_strides_of_dimensions_with_one_entry_mean_nothing():
    from patchaugnet_amd.attention import paged_append, paged_attention
    q, k, v = _inputs(1, 40, 1, 1, 32, BF16, seed=2)
    kp, vp, table = _cache(k, v, 40, [40], spare=0)
    want = paged_attention(q, kp, vp, table, _i([40]))

    def odd(t):
        return t.as_strided(t.shape, tuple(s if n > 1 else 13 for s, n in zip(t.stride(), t.shape)))

    assert odd(kp).stride(0) == 13 and odd(kp).is_contiguous()
    assert torch.equal(want, paged_attention(odd(q), odd(kp), odd(vp), table, _i([40])))
    paged_append(odd(v[:, 3:4]), odd(k[:, 3:4]), odd(kp), odd(vp), table, _i([7]))
    assert torch.equal(kp[0, 7], v[0, 3]) and torch.equal(vp[0, 7], k[0, 3])


def test_append_of_more_pieces_than_threads():
    """2^31 pieces of 16 bytes and more, of one expanded row: all but the last tokens lie in front of the table."""
    from patchaugnet_amd.attention import paged_append
    T, Hk, D = (1 << 27) + 5, 8, 16
    k = torch.randn(1, 1, Hk, D, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(BF16)
    kp, vp = (torch.zeros(2, 4, Hk, D, dtype=BF16, device="cuda") for _ in range(2))
    paged_append(k.expand(1, T, Hk, D), (-k).expand(1, T, Hk, D), kp, vp, _i([[1, 0]]), _i([3 - T]))
    want = torch.zeros_like(kp)
    want[1, :3] = k[0]
    assert torch.equal(kp, want) and torch.equal(vp, -want)


def test_refused_pools_are_not_copied():
    from patchaugnet_amd.attention import paged_append, paged_attention
    q, k, v = _inputs(1, 16, 2, 2, 32, BF16)
    flat = torch.zeros(4096 * 16 * 2 * 32 + 8, dtype=BF16, device="cuda")
    shifted = flat[1:-7].view(4096, 16, 2, 32)
    skew = torch.zeros(4096, 16, 2, 33, dtype=BF16, device="cuda")[..., 1:]
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    for pool in (shifted, skew):
        for call in (lambda: paged_attention(q, pool, pool, _i([[0]]), _i([16])), lambda: paged_append(k, v, pool, pool, _i([[0]]), _i([0]))):
            with pytest.raises(ValueError, match="16 bytes"):
                call()
    assert torch.cuda.max_memory_allocated() - before < flat.numel()


def test_gradients_do_not_read_stale_rows():
    """window_attention over rows of a pool, then an append into it: the backward pass says so instead of using the new rows."""
    from patchaugnet_amd.attention import paged_append, window_attention
    q, k, v = _inputs(1, 32, 2, 2, 32, BF16)
    kp, vp, table = _cache(k, v, 32, [32], spare=0)
    leaf = q.unsqueeze(1).clone().requires_grad_()
    out = window_attention(leaf, kp, vp, q_start=_i([31]))
    paged_append(k[:, :1], v[:, :1], kp, vp, table, _i([5]))
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    with torch.inference_mode():
        paged_append(k[:, :1], v[:, :1], kp.clone(), vp.clone(), table, _i([5]))
