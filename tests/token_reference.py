"""Plain 64-bit layer norm and attention with element-wise error bounds.

Each reference returns (value, bound) pairs.  A bound is the first-order worst case
of the operators' documented arithmetic, times SLACK for the second-order terms:
fp32 sums and products (unit roundoff F), the outputs rounded once to their type
(unit roundoff U), and for 16-bit types the probabilities and dS rounded to that
type before they multiply (U again, plus the type's smallest step where it is
fp16)."""
import torch

F = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}
STEP = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float64: 0.0}
SLACK = 1.25
ACC = 64  # longest chain of additions of a row sum: 32 in a thread, then a tree


def layer_norm(x, w, b, eps, dy=None):
    """x (R, C) and dy of the dtype under test -> dict of (value, bound)."""
    u = U[x.dtype]
    f = 2.0 ** -53 if x.dtype == torch.float64 else F
    uw = U[w.dtype] if w is not None else u
    R, C = x.shape
    x = x.double()
    wd = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = c.square().mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = c * rstd
    # the mean's error shifts every xh; the variance picks it up squared only
    e_mean = ACC * f * x.abs().mean(1, keepdim=True)
    e_xh = rstd * (e_mean + 2 * f * (x.abs() + mean.abs())) + xh.abs() * (ACC + 8) * f
    # the centred squares inherit 2 |c| e_c: relative 2 e_c / sigma on the variance
    e_c = e_mean + 2 * f * (x.abs() + mean.abs())
    rel_rstd = (c.abs() * e_c).mean(1, keepdim=True) * rstd.square()
    e_xh = e_xh + xh.abs() * rel_rstd
    y = xh * wd + bd
    step = STEP[torch.float16] if u == 2.0 ** -11 else 0.0
    out = {"y": (y, SLACK * (u * y.abs() + e_xh * wd.abs() + 4 * f * ((xh * wd).abs() + bd.abs())) + step)}
    if dy is not None:
        g = dy.double()
        gu = g * wd
        m1 = gu.mean(1, keepdim=True)
        m2 = (gu * xh).mean(1, keepdim=True)
        dx = rstd * (gu - m1 - xh * m2)
        e1 = ACC * f * gu.abs().mean(1, keepdim=True)
        e2 = ACC * f * (gu * xh).abs().mean(1, keepdim=True) + (gu.abs() * e_xh).mean(1, keepdim=True)
        mag = gu.abs() + m1.abs() + (xh * m2).abs()
        e = rstd * (e1 + xh.abs() * e2 + e_xh * m2.abs() + 6 * f * mag) + dx.abs() * (rel_rstd + (ACC + 8) * f)
        out["dx"] = (dx, SLACK * (u * dx.abs() + e) + step)
        n = 512 + R / 128  # a thread's rows, the groups of a block, the blocks' strands
        dw, db = (g * xh).sum(0), g.sum(0)
        out["dw"] = (dw, SLACK * (uw * dw.abs() + n * f * (g * xh).abs().sum(0) + (g.abs() * e_xh).sum(0)) + step)
        out["db"] = (db, SLACK * (uw * db.abs() + n * f * g.abs().sum(0)) + step)
    return out


def attend(q, k, v, seen, scale, do=None):
    """One head: q (n, D), k, v (m, D) of the dtype under test, seen (n, m) bool -> dict of (value, bound).

    Only tokens that `seen` lets through are looked at, so masked places may hold anything."""
    dtype = q.dtype
    u, step = U[dtype], STEP[dtype]
    n, d = q.shape
    zero = torch.zeros((), dtype=torch.float64, device=q.device)
    use_k, use_q = seen.any(0), seen.any(1)
    q = torch.where(use_q[:, None], q.double(), zero)
    k, v = torch.where(use_k[:, None], k.double(), zero), torch.where(use_k[:, None], v.double(), zero)
    s = scale * (q @ k.T)
    top = s.masked_fill(~seen, -1e300).amax(1, keepdim=True) if k.shape[0] else torch.zeros(n, 1, dtype=torch.float64, device=q.device)
    p = torch.where(seen, torch.exp(s - torch.where(use_q[:, None], top, zero)), zero)
    total = p.sum(1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    m = k.shape[0]
    # a score's error is a probability's relative error; the row's own sum and its logarithm add theirs
    e_s = scale * (d + 4) * F * (q.abs() @ k.abs().T) + 8 * F * (s.abs() + top.abs().clamp(max=1e30) + 8)
    e_row = torch.where(seen, p * e_s, zero).sum(1, keepdim=True) + (m / 8 + 64) * F
    rel = e_s + e_row
    o = p @ v
    a = p @ v.abs()
    e_o = (p * rel) @ v.abs() + u * a + step * v.abs().sum(0)[None] + (m / 8 + 64) * F * a
    out = {"o": (o, SLACK * (e_o + u * o.abs() + step))}
    if do is not None:
        g = torch.where(use_q[:, None], do.double(), zero)
        gmax = g.abs().max() if g.numel() else zero
        dv = p.T @ g
        a = p.T @ g.abs()
        e_dv = (p * rel).T @ g.abs() + u * a + step * g.abs().sum(0)[None] + (n / 8 + 64) * F * a
        out["dv"] = (dv, SLACK * (e_dv + u * dv.abs() + step))
        dp = g @ v.T
        delta = (g * o).sum(1, keepdim=True)
        ds = p * (dp - delta)
        e_delta = (g.abs() * (e_o + u * o.abs() + step)).sum(1, keepdim=True) + (d + 4) * F * (g * o).abs().sum(1, keepdim=True)
        e_ds = p * (rel * (dp - delta).abs() + (d + 4) * F * (g.abs() @ v.abs().T) + e_delta + 4 * F * (dp.abs() + delta.abs()))
        # fp16 dS is scaled by a power of two that brings the largest |dO| to [1, 2): its step scales back
        e_ds = torch.where(seen, e_ds + u * ds.abs() + step * 2 * gmax, zero)
        for name, x, e, b in (("dq", ds, e_ds, k), ("dk", ds.T, e_ds.T, q)):
            val = scale * (x @ b)
            err = scale * (e @ b.abs() + (x.shape[1] / 8 + 64) * F * (x.abs() @ b.abs()))
            out[name] = (val, SLACK * (err + u * val.abs() + step))
    return out


def packed(q, k, v, offsets, offsets_k, causal, scale, do=None):
    """Packed clouds, heads grouped: dict of (value, bound), laid out as the operator's."""
    T, H, D = q.shape
    Tk, Hk, _ = k.shape
    names = {"o": (T, H, D)}
    if do is not None:
        names.update(dq=(T, H, D), dk=(Tk, Hk, D), dv=(Tk, Hk, D))
    out = {n: tuple(torch.zeros(s, dtype=torch.float64, device=q.device) for _ in range(2)) for n, s in names.items()}
    for i in range(len(offsets) - 1):
        rows = slice(int(offsets[i]), int(offsets[i + 1]))
        keys = slice(int(offsets_k[i]), int(offsets_k[i + 1]))
        n, m = rows.stop - rows.start, keys.stop - keys.start
        if n == 0:
            continue
        seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril(m - n)
        for h in range(H):
            kh = h // (H // Hk)
            r = attend(q[rows, h], k[keys, kh], v[keys, kh], seen, scale, None if do is None else do[rows, h])
            for j in range(2):
                out["o"][j][rows, h] = r["o"][j]
                if do is not None:
                    out["dq"][j][rows, h] = r["dq"][j]
                    out["dk"][j][keys, kh] += r["dk"][j]
                    out["dv"][j][keys, kh] += r["dv"][j]
    return out


def cached(q, k, v, lengths, scale):
    out = tuple(torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    group = q.shape[1] // k.shape[2]
    for n, length in enumerate(lengths):
        length = min(max(int(length), 0), k.shape[1])
        for h in range(k.shape[2]):
            r = slice(h * group, (h + 1) * group)
            seen = torch.ones(group, length, dtype=torch.bool, device=q.device)
            got = attend(q[n, r], k[n, :length, h], v[n, :length, h], seen, scale)
            for j in range(2):
                out[j][n, r] = got["o"][j]
    return {"o": out}


def check(got, ref, name=""):
    """got (tensor) against (value, bound)."""
    value, bound = ref
    assert got.shape == value.shape, (name, got.shape, value.shape)
    off = (got.double() - value).abs()
    bad = ~(off <= bound)
    if bad.any():
        i = int(torch.where(bad, torch.nan_to_num(off / bound, nan=1e30), torch.zeros_like(off)).argmax())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside their bound; worst at {i}: got "
                             f"{got.flatten()[i].item()!r}, want {value.flatten()[i].item()!r} +- {bound.flatten()[i].item():.3g}")
