"""Plain float64 forms of the attention operators and of the 4-bit product on the CPU, with bounds of what rounding
can do to a kernel that holds scores, statistics and sums in 32-bit floats.

Bounds, with u = half a step of the element type relative to a value (finfo.eps / 2) and e = 2^-24 the same of float32:
a score is a sum of d products in float32, scaled and turned into a power of two, so it is off by at most
  ds <= (d + 4) e * scale * sum |q k|  (largest over the visible keys) + 8 e * max |s|,
which moves a weight by the factor exp(ds) and its normalisation by as much; sums over n keys add (n + 16) e of the sum of
magnitudes (exponentials and logarithms: a few e).  Where weights are rounded to the element type before a product
they add u, and, where that type is float16, half a step of its subnormal numbers (2^-25) for each weight, since a
weight (at most 1) or a weight's gradient below 2^-14 is rounded to a multiple of 2^-24.  The result's own rounding adds u
of the result.
"""
import torch

E32 = 2.0 ** -24


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def quantum(dtype) -> float:
    """Half a step of the type's subnormal numbers, where weights are rounded to it."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2 if dtype != torch.float32 else 0.0


def visible(nq, nk, window, sinks):
    p = torch.arange(nq)[:, None] + nk - nq
    j = torch.arange(nk)[None, :]
    seen = (j <= p)
    if window:
        seen &= (p - j < window) | (j < sinks)
    return seen


def attention(q, k, v, window=0, sinks=0, scale=None, rounded_weights=True):
    """One sequence: q [nq, h, d], k and v [nk, hk, d] (any type, any device) -> dict of float64: out, lse, their bounds
    (tol_out, tol_lse) and what the gradients need."""
    u, least = half_step(q.dtype), quantum(q.dtype)
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    nq, h, d = q.shape
    nk, hk, _ = k.shape
    scale = d ** -0.5 if scale is None else scale
    seen = visible(nq, nk, window, sinks)
    kk = k.repeat_interleave(h // hk, 1).transpose(0, 1)      # [h, nk, d]
    vv = v.repeat_interleave(h // hk, 1).transpose(0, 1)
    qq = q.transpose(0, 1)
    neg = torch.tensor(float("-inf"), dtype=torch.float64)
    s = torch.where(seen, scale * qq @ kk.transpose(1, 2), neg)
    mag = torch.where(seen, abs(scale) * qq.abs() @ kk.abs().transpose(1, 2), torch.zeros(()).double())
    lse = torch.logsumexp(s, -1) if nk else torch.full((h, nq), float("-inf")).double()
    empty = ~seen.any(-1)
    p = torch.where(seen & ~empty[:, None], torch.exp(s - lse[..., None]), torch.zeros(()).double())
    vsafe = torch.where(torch.isfinite(vv), vv, torch.zeros(()).double())
    out = p @ vsafe
    n = seen.sum(-1).double()
    big = mag.amax(-1) if nk else torch.zeros(h, nq).double()
    ds = (d + 4) * E32 * big + 8 * E32 * big
    weight = 2 * ds + (n + 16) * E32                                     # relative error of a weight
    pv = p @ vsafe.abs()
    tol = u * out.abs() + ((u if rounded_weights and u > E32 else 0.0) + weight[..., None]) * pv * 1.01
    if rounded_weights:
        tol = tol + least * (seen & ~empty[:, None]).double() @ vsafe.abs()
    tol_lse = ds + (n + 16) * E32 + 4 * E32 * lse.abs().nan_to_num(posinf=0, neginf=0)
    t = lambda x: x.transpose(0, 1)
    return dict(out=t(out), lse=t(lse), tol_out=t(tol), tol_lse=t(tol_lse), p=p, weight=weight, qq=qq, kk=kk, vv=vv,
                scale=scale, u=u, least=least * seen, h=h, hk=hk, n=n)


def gradients(r, dout):
    """Gradients of `attention`'s r for dout [nq, h, d], with bounds: dict of dq, dk, dv, tol_dq, tol_dk, tol_dv.

    D = <dout, out> is taken from the rounded out: off by |dout| . tol_out.  dS = P (dP - D) is rounded to the element type
    (u), and carries the weight's error and those of dP ((d + 2) e of its magnitudes) and D."""
    p, weight, qq, kk, vv, scale, u = (r[x] for x in ("p", "weight", "qq", "kk", "vv", "scale", "u"))
    do = dout.detach().cpu().double().transpose(0, 1)
    d = do.shape[-1]
    ur = u if u > E32 else 0.0
    dp = do @ vv.transpose(1, 2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    err_dp = (d + 2) * E32 * (do.abs() @ vv.abs().transpose(1, 2))
    out, tol_out = r["out"].transpose(0, 1), r["tol_out"].transpose(0, 1)
    err_delta = (do.abs() * (tol_out + (d + 2) * E32 * out.abs())).sum(-1, keepdim=True)
    w2 = 2 * weight[..., None] + 8 * E32
    err_ds = (ur + w2) * ds.abs() + p * (err_dp + err_delta) * 1.01 + r["least"]
    nq = qq.shape[1]
    sums = (nq * r["h"] / r["hk"] + 16) * E32                            # sums over the queries of a group's heads
    fold = lambda x: x.reshape(r["hk"], r["h"] // r["hk"], *x.shape[1:]).sum(1)
    res = {}
    dq = scale * ds @ kk
    res["dq"], res["tol_dq"] = dq, u * dq.abs() + abs(scale) * (err_ds + (r["n"][:, None] + 16) * E32 * ds.abs()) @ kk.abs() * 1.01
    dk = fold(scale * ds.transpose(1, 2) @ qq)
    res["dk"], res["tol_dk"] = dk, u * dk.abs() + abs(scale) * fold((err_ds + sums * ds.abs()).transpose(1, 2) @ qq.abs()) * 1.01
    dv = fold(p.transpose(1, 2) @ do)
    res["dv"], res["tol_dv"] = dv, u * dv.abs() + fold(((ur + w2 + sums) * p + r["least"]).transpose(1, 2) @ do.abs()) * 1.01
    return {n: x.transpose(0, 1) for n, x in res.items()}


def check(name, got, want, tol):
    """|got - want| <= tol (plus the smallest numbers of the type), infinities and NaN in the same places."""
    tiny = torch.finfo(got.dtype).tiny * (1 if got.dtype != torch.float16 else 2.0 ** -10)
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    ok = torch.where(torch.isfinite(want), (got - want).abs() <= tol + tiny, (got == want) | (got.isnan() & want.isnan()))
    if not bool(ok.all()):
        bad = (~ok).nonzero()[0].tolist()
        worst = ((got - want).abs() / (tol + tiny)).nan_to_num(nan=float("inf")).max()
        raise AssertionError(f"{name}: {int((~ok).sum())} of {ok.numel()} off, first at {bad}: "
                             f"{got[tuple(bad)]} for {want[tuple(bad)]}, worst {worst:.3g} of the bound")


def q4_weights(packed, scales, zeros, cols, group):
    """(w, magnitude of what the kernel sums for a unit x) in float64, [rows, cols]."""
    q = torch.stack((packed.cpu() & 15, packed.cpu() >> 4), 2).reshape(packed.shape[0], -1)[:, :cols].double()
    g = torch.arange(cols) // group
    z = zeros.cpu().double()[:, g] if zeros is not None else torch.full_like(q, 8.0)
    s = scales.cpu().double()[:, g]
    return (q - z) * s, (32 + q + z) * s.abs()
