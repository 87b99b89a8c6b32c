"""64-bit reference of the score-modified attention, with first-order error bounds.

Plain torch in float64, one dense score matrix per call, on whatever device the operands are on;
test infrastructure only.  The formulas are those of ``SM120ScoreAttentionDesc`` in
include/sm120_c_interface.h.

Error bounds.  ``u`` is half a step of the operands' type relative to the value (``finfo.eps / 2``);
fp32 additions in the tensor cores may truncate, so each costs up to 2^-23 of the running magnitude.

  score      |d x| <= D 2^-23 scale sum|q||k|; the cap does not enlarge it (|tanh'| <= 1) and adds 2^-21 of the cap;
             the bias adds 2^-22 of itself and the final sum and the change to base 2 add 2^-21 |z|
  weights    relative error 2 |d z| + 2^-20 (exponential, denominator) =: d, plus u for the rounding before the
             second product
  out        (u + 2 d) sum P|v| + n 2^-23 sum P|v| / 16 + u |out|
  dx         (u + d) |dx| + P (|d dP| + |d Delta|), with |d dP| <= D 2^-23 sum|do||v| and
             |d Delta| <= sum|do| |d out| + D 2^-23 sum|do||out|
  gradients  the bound of dx (or of P) through the absolute second factor, plus the final rounding
float16 has a smallest step of 2^-24: weights and dx below its normal range are off by 2^-25 absolutely.  The other
types have fp32's range, whose smallest normal number is 2^-126: a weight below it may come out as 0, and with it a
gradient of weight times |dP - Delta|.
"""
import math

import torch


def visible(batch, seq_q, seq_k, *, causal=False, document_offsets=None, prefix_lengths=None, device="cpu"):
    """[batch, seq_q, seq_k] truth values: does the query see the key?"""
    i = torch.arange(seq_q, device=device)[:, None] + (seq_k - seq_q)
    j = torch.arange(seq_k, device=device)[None, :]
    seen = torch.ones((batch, seq_q, seq_k), dtype=torch.bool, device=device)
    for b in range(batch):
        if causal:
            bound = j <= i
            if prefix_lengths is not None:
                bound = bound | (j < int(prefix_lengths[b]))
            seen[b] &= bound
        if document_offsets is not None:
            same = torch.zeros((seq_q, seq_k), dtype=torch.bool, device=device)
            offs = [min(max(int(o), 0), seq_k) for o in document_offsets[b]]
            for lo, hi in zip(offs, offs[1:]):
                same |= (i >= lo) & (i < hi) & (j >= lo) & (j < hi)
            seen[b] &= same
    return seen


def attention(q, k, v, *, scale=None, softcap=None, slopes=None, seen=None, grad_out=None):
    """q [B, H, Sq, D], k and v [B, Hk, Sk, D] -> dict of float64 results and bounds of their errors
    (``out``, ``lse`` and, with ``grad_out``, ``dq``, ``dk``, ``dv``; the bound of x is ``x_tol``)."""
    dtype, f64 = q.dtype, torch.float64
    u = torch.finfo(dtype).eps / 2
    b, h, sq, d = q.shape
    hk, sk = k.shape[1], k.shape[2]
    g = h // hk
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    q = q.to(f64)
    # content of keys that nobody sees does not count
    used = seen.any(1)[:, None, :, None] if seen is not None else torch.ones((), dtype=torch.bool, device=q.device)
    k, v = (torch.where(used, t.to(f64), 0.0) for t in (k, v))
    some = seen.any(2)[:, None, :, None] if seen is not None else used
    q = torch.where(some, q, 0.0)
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    eps, n = 2.0 ** -23, max(sk, 1)
    x = q @ kk.transpose(-1, -2) * scale
    dz = d * eps * abs(scale) * (q.abs() @ kk.abs().transpose(-1, -2))
    curve = torch.zeros_like(x)
    z = x
    if softcap:
        curve = torch.tanh(x / softcap)
        z = softcap * curve
        dz = dz + 4 * eps * softcap
    if slopes is not None:
        away = ((torch.arange(sq, device=q.device)[:, None] + (sk - sq)) - torch.arange(sk, device=q.device)[None, :]).abs().to(f64)
        bias = slopes.to(f64)[None, :, None, None] * away
        z = z - bias
        dz = dz + 2 * eps * bias.abs()
    dz = dz + 4 * eps * z.abs()
    if seen is not None:
        z = z.masked_fill(~seen[:, None], -math.inf)
        dz = dz.masked_fill(~seen[:, None], 0.0)
    lse = torch.logsumexp(z, -1) if sk else torch.full((b, h, sq), -math.inf, dtype=f64, device=q.device)
    p = torch.exp(z - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    dlse = (p * dz).sum(-1, keepdim=True)
    dp_rel = dz + dlse + 8 * eps
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    out = p @ vv
    mass = p @ vv.abs()
    out_tol = ((p * (u + 2 * dp_rel)) @ vv.abs() + n / 16 * eps * mass + tiny * vv.abs().sum(-2, keepdim=True) * some + u * out.abs() + tiny) * 1.01
    res = {"out": out, "out_tol": out_tol, "lse": lse,
           "lse_tol": (dlse[..., 0] + 4 * eps + 2 * eps * torch.where(lse == -math.inf, 0.0, lse.abs()) + n / 32 * eps) * 1.01}
    if grad_out is None:
        return res
    do = torch.where(some, grad_out.to(f64), 0.0)
    back = do @ vv.transpose(-1, -2)
    delta = (do * out).sum(-1, keepdim=True)
    dx = p * (back - delta) * (1 - curve * curve)
    back_tol = d * eps * (do.abs() @ vv.abs().transpose(-1, -2))
    delta_tol = (do.abs() * out_tol).sum(-1, keepdim=True) + d * eps * (do.abs() * out.abs()).sum(-1, keepdim=True)
    dx_tol = (u + dp_rel + 8 * eps) * dx.abs() + p * (back_tol + delta_tol + 4 * eps * (back.abs() + delta.abs())) \
        + (tiny + 2.0 ** -126 * (back - delta).abs()) * (p > 0)
    if softcap:
        dx_tol = dx_tol + p * (back - delta).abs() * 2 * (dz / softcap + 8 * eps)
    p_tol = p * (u + dp_rel) + tiny * (p > 0)

    def heads(t):
        return t.view(b, hk, g, sk, d).sum(2)

    rows = g * sq
    res["dq"] = dx @ kk * scale
    res["dq_tol"] = (abs(scale) * ((dx_tol + n / 16 * eps * dx.abs()) @ kk.abs()) + u * res["dq"].abs() + tiny) * 1.01
    res["dk"] = heads(dx.transpose(-1, -2) @ q) * scale
    res["dk_tol"] = (abs(scale) * heads((dx_tol + rows / 16 * eps * dx.abs()).transpose(-1, -2) @ q.abs()) + u * res["dk"].abs() + tiny) * 1.01
    res["dv"] = heads(p.transpose(-1, -2) @ do)
    res["dv_tol"] = (heads((p_tol + rows / 16 * eps * p).transpose(-1, -2) @ do.abs()) + u * res["dv"].abs() + tiny) * 1.01
    return res


def token_attention(q, k, v, lengths, *, prefix_k=None, prefix_v=None, scale=None, softcap=None, slopes=None):
    """The single-token form, request by request through ``attention``: q [B, H, D], caches [B, Hk, S, D]."""
    rows = []
    for b, length in enumerate(int(x) for x in lengths):
        length = min(max(length, 0), k.shape[2])
        keys, values = k[b, :, :length], v[b, :, :length]
        if prefix_k is not None:
            keys, values = torch.cat([prefix_k, keys], 1), torch.cat([prefix_v, values], 1)
        rows.append(attention(q[b][None, :, None], keys[None], values[None], scale=scale, softcap=softcap, slopes=slopes))
    return {name: torch.cat([r[name][:, :, 0] for r in rows]) for name in rows[0]}
