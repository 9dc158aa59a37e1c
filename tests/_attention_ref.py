"""64-bit statement of the windowed attention and its gradients, with elementwise error bounds for a kernel that holds sums in 32 bits.

Bounds, to first order.  u: half a step of the tensors' type (torch.finfo(t).eps / 2), w = 2^-24.
  scores      e_ij = w (D a_ij + 4 |s_ij|), a_ij = scale sum_d |q_id k_jd|: D products summed, the scale, the exponent's argument, the reference value
  weights     P_ij (1 + 2 E_i + r),  E_i = max_j e_ij + w (M + 32): the sum's terms, exp2, the quotient; r = u where 16-bit operands round P, else 0
  out         u |o| + sum_j P_ij (2 E_i + r) |v_j| + w (M + 32) sum_j P_ij |v_j|
  flush       v_exp_f32 gives 0 for results below F = 2^-126, and a product below F adds 0 to a 32-bit sum: P_ij is off by up to F in absolute terms
              (times |v_j|, |do_i|, |dP_ij - delta_i| |k_j| or |q_i| where it is used), and every term of a sum by F
  dS          |dS| (2 E_i + r) + P_ij (c_i + w D sum_d |do_id v_jd|), c_i = u_o sum |do_id o_id| + error of out . |do| + w D sum |do_id o_id|
"""
import torch

W = 2.0 ** -24
F = 2.0 ** -126


def seen(N, M, left, right, sinks, length, start, device="cpu"):
    """(N, M) truth values: query i at start + i sees key j."""
    p = start + torch.arange(N, device=device).view(-1, 1)
    j = torch.arange(M, device=device).view(1, -1)
    ok = (p < length) & (j < length)
    if right is not None:
        ok = ok & (j <= p + right)
    if left is not None:
        ok = ok & ((j >= p - left) | (j < sinks))
    return ok


def reference(q, k, v, left, right, sinks, scale=None, lengths=None, starts=None, dout=None):
    """(values, bounds): dicts with out and, given dout, dq, dk, dv in 64 bits, shaped like the inputs."""
    B, N, H, D = q.shape
    M, Hk = k.shape[1], k.shape[2]
    u = torch.finfo(q.dtype).eps / 2
    r = u if q.dtype != torch.float32 else 0.0
    scale = D ** -0.5 if scale is None else scale
    names = ["out"] + (["dq", "dk", "dv"] if dout is not None else [])
    like = {"out": q, "dq": q, "dk": k, "dv": v}
    val = {n: torch.zeros(like[n].shape, dtype=torch.float64, device=q.device) for n in names}
    tol = {n: torch.zeros_like(val[n]) for n in names}
    for b in range(B):
        ln = M if lengths is None else int(min(max(int(lengths[b]), 0), M))
        st = 0 if starts is None else int(min(max(int(starts[b]), 0), M))
        ok = seen(N, M, left, right, sinks, ln, st, q.device)
        rows = ok.any(1)
        for h in range(H):
            g = h // (H // Hk)
            Q, K, V = q[b, :, h].double(), k[b, :, g].double(), v[b, :, g].double()
            Q = torch.where(rows[:, None], Q, 0.0)
            live = (torch.arange(M, device=q.device) < ln)[:, None]
            K, V = torch.where(live, K, 0.0), torch.where(live, V, 0.0)
            s = scale * (Q @ K.t().contiguous())
            a = scale * (Q.abs() @ K.abs().t().contiguous())
            s = s.masked_fill(~ok, float("-inf"))
            P = torch.softmax(s, 1).nan_to_num(nan=0.0)
            e = torch.where(ok, W * (D * a + 4 * s.abs()), 0.0)
            E = e.amax(1, keepdim=True) + W * (M + 32) if M else torch.zeros(N, 1, dtype=torch.float64, device=q.device)
            o = P @ V
            po = P @ V.abs()
            o_err = po * (2 * E + r + W * (M + 32)) + F * (V.abs().sum(0, keepdim=True) + M)
            val["out"][b, :, h] = o
            tol["out"][b, :, h] = u * o.abs() + o_err
            if dout is None:
                continue
            G = torch.where(rows[:, None], dout[b, :, h].double(), 0.0)
            dP, dPa = G @ V.t().contiguous(), G.abs() @ V.abs().t().contiguous()
            delta = (G * o).sum(1, keepdim=True)
            c = (G.abs() * (u * o.abs() + o_err + W * D * o.abs())).sum(1, keepdim=True)
            dS = P * (dP - delta)
            eS = dS.abs() * (2 * E + r + 4 * W) + P * (c + W * D * dPa) + F * ((dP - delta).abs() + 1)
            eP = P * (2 * E + r) + F
            n = W * (max(N, M) * H + 32)                       # 32-bit sums over rows of all heads of a group, or over keys
            val["dq"][b, :, h] = scale * (dS @ K)
            tol["dq"][b, :, h] = scale * (eS @ K.abs() + n * (dS.abs() @ K.abs()))
            val["dk"][b, :, g] += scale * (dS.t().contiguous() @ Q)
            tol["dk"][b, :, g] += scale * (eS.t().contiguous() @ Q.abs() + n * (dS.abs().t().contiguous() @ Q.abs()))
            val["dv"][b, :, g] += P.t().contiguous() @ G
            tol["dv"][b, :, g] += eP.t().contiguous() @ G.abs() + n * (P.t().contiguous() @ G.abs())
    tiny = torch.finfo(q.dtype).smallest_normal * u * 2        # half a step among the type's subnormal numbers, and one for the operands
    for n in names:
        if n != "out":
            tol[n] += u * val[n].abs()
        tol[n] += tiny * (1 if n == "out" else max(N, M) * 8) + F * max(N, M) * H
    return val, tol


def close(got, val, tol, what):
    assert got.shape == val.shape, (what, got.shape, val.shape)
    err = (got.double() - val).abs()
    bad = ~(err <= tol)                                         # NaN is bad
    assert not bad.any(), (what, int(bad.sum()), "of", bad.numel(), "largest error / bound", float((err / tol.clamp_min(1e-300)).max()))
