"""The decoder attention's definition in 64 bits, with the bound its tests use."""
import math

import torch

U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def reference(q, k, v, scale=None, softcap=0.0, slopes=None, q_pos=None, k_pos=None, q_segment=None, k_segment=None,
              k_len=None, dout=None):
    """A dict in fp64: ``out``, ``lse`` and ``out_abs`` = sum P |V|; with ``dout`` also ``dq``, ``dk``, ``dv`` and
    ``dslopes [B, Nq, H]`` and the bound of each before its own last rounding (``*_tol``).  Values at
    masked pairs take no part, whatever they are.  Loops over batch entries and heads."""
    B, Nq, H, D = q.shape
    Nk, G = k.shape[1], k.shape[2]
    dev = q.device
    scale = D ** -0.5 if scale is None else scale
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=dev)  # noqa: E731
    r = dict(out=z(B, Nq, H, D), lse=torch.full((B, H, Nq), -math.inf, dtype=torch.float64, device=dev),
             out_abs=z(B, Nq, H, D))
    if dout is not None:
        h16 = half_step(q.dtype)
        e = score_error(q, k, scale, softcap, slopes, q_pos, k_pos)
        for n, shape in (("dq", (B, Nq, H, D)), ("dk", (B, Nk, G, D)), ("dv", (B, Nk, G, D)), ("dslopes", (B, Nq, H))):
            r[n], r[n + "_tol"] = z(*shape), z(*shape)
    for b in range(B):
        ok = torch.ones(Nq, Nk, dtype=torch.bool, device=dev)
        if k_len is not None:
            ok[:, max(0, min(Nk, int(k_len[b]))):] = False
        if q_segment is not None:
            ok &= (q_segment[b][:, None] == k_segment[b][None]) & (q_segment[b][:, None] >= 0)
        rows, cols = ok.any(1), ok.any(0)
        dist = None
        if slopes is not None:
            dist = (q_pos[b].double()[:, None] - k_pos[b].double()[None]).square().sum(-1).sqrt()
            dist = torch.where(ok, dist, torch.zeros_like(dist))
        for h in range(H):
            g = h // (H // G)
            Q = torch.where(rows[:, None], q[b, :, h].double(), z(1))
            K, V = (torch.where(cols[:, None], t[b, :, g].double(), z(1)) for t in (k, v))
            x = scale * (Q @ K.T)
            s = softcap * torch.tanh(x / softcap) if softcap else x
            t = s / softcap if softcap else None
            if dist is not None:
                sl = slopes[h] if slopes.dim() == 1 else slopes[b, :, h]
                s = s - sl.double().reshape(-1, 1) * dist
            s = torch.where(ok, s, torch.full_like(s, -math.inf))
            lse = torch.logsumexp(s, 1)
            p = torch.where(ok, torch.exp(s - torch.where(rows, lse, z(1))[:, None]), z(1))
            r["lse"][b, h] = lse
            r["out"][b, :, h] = p @ V
            r["out_abs"][b, :, h] = p @ V.abs()
            if dout is None:
                continue
            dO = torch.where(rows[:, None], dout[b, :, h].double(), z(1))
            dp = dO @ V.T
            delta = (p * dp).sum(1, keepdim=True)
            ds = p * (dp - delta)
            dx = ds * (1 - t * t) if softcap else ds
            r["dq"][b, :, h] = scale * dx @ K
            r["dk"][b, :, g] += scale * dx.T @ Q
            r["dv"][b, :, g] += p.T @ dO
            # Bounds.  A weight is off by 2 e (score and log-sum-exp); dP by D u of its products; delta
            # by h of |dO| |out| (out is rounded) and D u; the cap's derivative by 16 u; dX and P are
            # rounded to the type once (h); sums over N terms by N u.
            row = p * (dO.abs() * r["out"][b, :, h].abs()).sum(1, keepdim=True)
            mag = p * (dO.abs() @ V.abs().T) + row
            off = 2 * e * ds.abs() + 16 * U * ds.abs() + (D + 8) * U * mag
            dx_off = (h16 + max(Nq, Nk) * U) * dx.abs() + off + h16 * row
            r["dq_tol"][b, :, h] = abs(scale) * dx_off @ K.abs()
            r["dk_tol"][b, :, g] += abs(scale) * dx_off.T @ Q.abs()
            r["dv_tol"][b, :, g] += (h16 + 2 * e + max(Nq, Nk) * U) * p.T @ dO.abs()
            if dist is not None:
                r["dslopes"][b, :, h] = -(ds * dist).sum(1)
                # delta's rounding cancels up to the error of sum P = 1
                r["dslopes_tol"][b, :, h] = ((off + Nk * U * mag + (2 * e + Nk * U) * h16 * row) * dist).sum(1) \
                    + (2 * e + Nk * U) * h16 * row.sum(1) * (p * dist).sum(1)
    return r


def score_error(q, k, scale, softcap, slopes, q_pos, k_pos):
    """Bound on the absolute error of a score in fp32: D products added in fp32 (D u of the sum of their
    magnitudes, at most |q| |k|), the cap (4 u per unit of cap: exponential, reciprocal and two
    roundings, each 2 u), the bias (the square root and its product, 8 u of slope * distance, the
    coordinates' differences 4 u) and the exponent's own roundings."""
    D = q.shape[-1]
    sc = D ** -0.5 if scale is None else abs(scale)
    qk = sc * q.double().norm(dim=-1).nan_to_num(0, 0, 0).max() * k.double().norm(dim=-1).nan_to_num(0, 0, 0).max()
    e = (D + 8) * U * float(qk)
    top = float(qk)
    if softcap:
        e += 16 * U * softcap
        top = min(top, softcap)
    if slopes is not None and q_pos.numel() and k_pos.numel():
        far = float((q_pos.abs().amax() + k_pos.abs().amax()) * 2)
        e += 16 * U * float(slopes.abs().max()) * far
        top += float(slopes.abs().max()) * far
    return e + 8 * U * top
