"""The training-layer operators in 64 bits, from their definitions, with bounds on what a computation in 32 bits (and its
roundings to the tensors' type) may differ by.  For the tests only."""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# half a step below the normal numbers; where the type has 32-bit range, weights below 2^-126 count as none, for up to 2^10 of them on values of up to 2^6
SMALLEST = {torch.bfloat16: 2.0 ** -110, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -110}


def close(got, want, slack):
    """|got - want| <= one rounding of want + slack, and the same values that are no numbers."""
    u = UNIT[got.dtype]
    got, want, slack = got.double().cpu(), want.double().cpu(), slack.double().cpu()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan())
    fine = want.isfinite()
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    off = (got - want).abs()[fine] - (u * want.abs() * (1 + 2 ** -6) + slack)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, f"{float(off.max())} beyond the bound, at {int(off.argmax())} of {off.numel()}"


# ---- norms around a block -----------------------------------------------------------------------------------------------------
def norm_parts(u, kind, eps):
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    rstd = (u.square().mean(-1, keepdim=True) + eps).rsqrt()
    return u * rstd, rstd


def block_norm(x, block, residual_scale, gate, exit_weight, exit_bias, entry_weight, entry_bias, kind, eps, **_):
    """(residual, normed) in 64 bits; gate already of a shape that broadcasts over x."""
    residual = x
    if block is not None:
        z = block
        if exit_weight is not None:
            z = norm_parts(z, kind, eps)[0] * exit_weight
            z = z if exit_bias is None else z + exit_bias
        residual = residual_scale * x + (z if gate is None else gate * z)
    normed = None
    if entry_weight is not None:
        normed = norm_parts(residual, kind, eps)[0] * entry_weight
        normed = normed if entry_bias is None else normed + entry_bias
    return residual, normed


def block_norm_grads(d_residual, d_normed, x, block, residual_scale, gate, exit_weight, exit_bias, entry_weight, entry_bias, kind, eps):
    """The gradients by their formulas: {name: (value, sum of the magnitudes that were added up for it)}.  What the residual's gradient
    goes into counts with the largest one of its row, and a sum of two with both: that is what their own rounding goes by."""
    def back(dn, n, rstd):
        d = dn - n * (dn * n).mean(-1, keepdim=True)
        return (d - dn.mean(-1, keepdim=True) if kind == "layer" else d) * rstd

    def over(t, like):
        lead = t.dim() - like.dim()
        t = t.sum(tuple(range(lead))) if lead else t
        keep = [i for i in range(like.dim()) if like.shape[i] == 1 and t.shape[i] != 1]
        return t.sum(keep, keepdim=True) if keep else t
    out = {}

    def summed(name, terms, like, sizes=None):
        out[name] = (over(terms, like), over((terms if sizes is None else sizes).abs(), like))
    n2 = rstd2 = z_size = None
    z, residual = block, x
    if block is not None:
        if exit_weight is not None:
            n2, rstd2 = norm_parts(block, kind, eps)
            z = n2 * exit_weight
            z = z if exit_bias is None else z + exit_bias
        z_size = z.abs() if exit_bias is None else (n2 * exit_weight).abs() + exit_bias.abs()
        residual = residual_scale * x + (z if gate is None else gate * z)
    dr = torch.zeros_like(x) if d_residual is None else d_residual
    if entry_weight is not None:
        dy = torch.zeros_like(x) if d_normed is None else d_normed
        n1, rstd1 = norm_parts(residual, kind, eps)
        dr = dr + back(dy * entry_weight, n1, rstd1)
        summed("entry_weight", dy * n1, entry_weight)
        if entry_bias is not None:
            summed("entry_bias", dy, entry_bias)
    size = dr.abs().amax(-1, keepdim=True).expand_as(dr)
    out["x"] = (residual_scale * dr, size)
    if block is not None:
        dz = dr if gate is None else dr * gate
        if gate is not None:
            summed("gate", dr * z, gate, size * z_size)
        if exit_weight is not None:
            summed("exit_weight", dz * n2, exit_weight, size * n2 * (1 if gate is None else gate))
            if exit_bias is not None:
                summed("exit_bias", dz, exit_bias, size * (1 if gate is None else gate))
            d_block = back(dz * exit_weight, n2, rstd2)
            out["block"] = (d_block, (rstd2 * (dz * exit_weight).abs().amax(-1, keepdim=True) * (1 + n2.abs().amax(-1, keepdim=True))).expand_as(dz))
        else:
            out["block"] = (dz, dz.abs().amax(-1, keepdim=True).expand_as(dz))
    return out


# ---- attention ------------------------------------------------------------------------------------------------------------------
def visible(batch, queries, keys, window, sinks, start, lengths):
    start = torch.full((batch,), keys - queries) if start is None else start.cpu().long()
    lengths = torch.full((batch,), keys) if lengths is None else lengths.cpu().long()
    p = start[:, None, None] + torch.arange(queries)[None, :, None]
    j = torch.arange(keys)[None, None, :]
    seen = (j < lengths[:, None, None]) & (j <= p)
    if window is not None:
        seen &= (p - j < window) | (j < sinks)
    return seen


def attention(q, k, v, window=None, sinks=0, scale=None, start=None, lengths=None, d_out=None, unit=0.0):
    """On the CPU, in 64 bits: {"out", "lse"} and with d_out {"dq", "dk", "dv"} too, each (value, bound beyond one rounding of the
    value), where weights and their gradients are rounded to numbers of unit roundoff `unit` before they meet the values."""
    q, k, v = (t.double().cpu().transpose(1, 2) for t in (q, k, v))
    shared = q.shape[1] // k.shape[1]
    scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    seen = visible(q.shape[0], q.shape[2], k.shape[2], window, sinks, start, lengths)[:, None]
    kx, vx = k.repeat_interleave(shared, 1), v.repeat_interleave(shared, 1)
    # (what is not seen by anyone is not read)
    anyone = seen.any(2)[..., None]
    kx, vx = torch.where(anyone, kx, 0.0), torch.where(anyone, vx, 0.0)
    s = (q @ kx.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, (s - torch.where(lse.isfinite(), lse, 0.0)[..., None]).exp(), 0.0)
    # a score is a sum of `size` products in 32 bits: that many units of the largest one, doubled for the exponential's own
    size = q.abs() @ kx.abs().transpose(2, 3) * scale
    wrong = 2.0 ** -24 * (2 * size.masked_fill(~seen, 0.0).amax(-1, keepdim=True) + 64)
    out = p @ vx
    r = {"out": (out, (unit + wrong) * (p @ vx.abs())), "lse": (lse, (wrong[..., 0] + 2.0 ** -20 * (1 + torch.where(lse.isfinite(), lse, 0.0).abs())))}
    if d_out is not None:
        do = d_out.double().cpu().transpose(1, 2)

        def kv(t):
            return t.unflatten(1, (-1, shared)).sum(2)
        dp, delta = do @ vx.transpose(2, 3), (do * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        # delta comes from the rounded answer; the rest of dS from 32 bits
        off = unit * ds.abs() + p * (2 * unit * (do.abs() * (out.abs() + p @ vx.abs())).sum(-1, keepdim=True) + 2 * wrong * (do.abs() @ vx.abs().transpose(2, 3) + delta.abs()))
        r["dv"] = (kv(p.transpose(2, 3) @ do), (unit + 2 * wrong.amax()) * kv(p.transpose(2, 3) @ do.abs()))
        r["dq"] = (scale * (ds @ kx), scale * (off @ kx.abs()))
        r["dk"] = (scale * kv(ds.transpose(2, 3) @ q), scale * kv(off.transpose(2, 3) @ q.abs()))
    return {n: (a, b) if n == "lse" else (a.transpose(1, 2), b.transpose(1, 2)) for n, (a, b) in r.items()}


# ---- AdamW ------------------------------------------------------------------------------------------------------------------------
def adamw(p, g, m, v, lr, betas, eps, weight_decay, step, grad_scale=1.0):
    b1, b2 = betas
    g = g * grad_scale
    m, v = m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)
    return p * (1 - lr * weight_decay) - lr / (1 - b1 ** step) * m / (v.sqrt() / math.sqrt(1 - b2 ** step) + eps), m, v
