"""Attention in 64 bits from its definition, with its gradients, and elementwise bounds of what a kernel may be off.

The bounds count roundings.  u = half a step of the data's type; g = d 2^-24, the bound of a d-long fp32 sum.
  scores     e_ij = g |scale| |q_i||k_j| plus 2^-22 of the score and its bias (the last steps of the epilogue), and with a
             tanh 2^-22 cap; an error e of a score changes its weight by the factor exp(e)
  out        u |out| (rounding of the result) + (u + e_max + 2^-18) P |V| (rounding of the weights to the data's type before
             they meet V; 2^-18: 2^-24 for each of the fp32 sums of weights, up to 64 of them one behind another)
  dV         u |dV| + (u + 2 e_max + 2^-18 + |lse| 2^-22) P^T |dO|
  dS         (u + 2 e_max + 2^-18 + |lse| 2^-22) |dS| + P (g |dO||V|^T + |dO|.E_out), E_out being the bound of out, because
             delta_i = dO_i . out_i uses the stored result
  dQ, dK     u |dQ| + |scale| (bound of dS) |K|, and so on
fp16 weights below its normal range are off by 2^-25 at most, which adds 2^-25 sum |V| and so on.
"""
import math

import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def visible(nq, nk, b, causal, prefix_lens, documents, q_documents, kv_lens, q_starts):
    """(b, nq, nk) truth values, and the positions of the queries (b, nq)."""
    see = torch.ones(b, nq, nk, dtype=torch.bool)
    at = torch.zeros(b, nq, dtype=torch.float64)
    for i in range(b):
        n = nk if kv_lens is None else min(max(int(kv_lens[i]), 0), nk)
        start = n - nq if q_starts is None else int(q_starts[i])
        at[i] = torch.arange(nq, dtype=torch.float64) + start
        col = torch.arange(nk)
        see[i] &= (col < n)[None, :]
        if causal:
            early = col[None, :] <= at[i][:, None]
            if prefix_lens is not None:
                early |= (col < int(prefix_lens[i]))[None, :]
            see[i] &= early
        if documents is not None:
            qd = documents if q_documents is None else q_documents
            see[i] &= (qd[i][:, None] == documents[i][None, :]) & (documents[i] >= 0)[None, :]
    return see, at


def reference(q, k, v, do=None, *, causal=False, scale=None, softcap=None, slopes=None, prefix_lens=None, documents=None,
              q_documents=None, kv_lens=None, q_starts=None):
    """dict with out, lse, dq, dk, dv (64 bits, on the data's device) and their bounds e_out, e_dq, ..."""
    dt, dev = q.dtype, q.device
    b, nq, hq, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    u, g = HALF_STEP[dt], d * 2.0**-24
    tiny = 2.0**-25 if dt == torch.float16 else 0.0
    scale = 1 / math.sqrt(d) if scale is None else scale
    cpu = [None if t is None else t.cpu() for t in (prefix_lens, documents, q_documents, kv_lens, q_starts)]
    see, at = (t.to(dev) for t in visible(nq, nk, b, causal, *cpu))
    r = {n: torch.zeros(b, nq if n in ("out", "dq") else nk, hq if n in ("out", "dq") else hk, d, dtype=torch.float64, device=dev)
         for n in ("out", "dq", "dk", "dv")}
    r.update({"e_" + n: torch.zeros_like(t) for n, t in r.items()})
    r["lse"] = torch.full((b, hq, nq), -math.inf, dtype=torch.float64, device=dev)
    r["e_lse"] = torch.zeros_like(r["lse"])
    col = torch.arange(nk, dtype=torch.float64, device=dev)
    for i in range(b):
        shown = see[i].any(0)  # keys that nobody sees may hold anything
        for h in range(hq):
            kv = h // (hq // hk)
            Q = q[i, :, h].detach().double()
            Q = torch.where(see[i].any(1)[:, None], Q, torch.zeros_like(Q))
            K = torch.where(shown[:, None], k[i, :, kv].detach().double(), 0.0)
            V = torch.where(shown[:, None], v[i, :, kv].detach().double(), 0.0)
            S = Q @ K.T * scale
            e = g * abs(scale) * (Q.abs() @ K.abs().T)
            t = torch.zeros_like(S)
            if softcap:
                t = torch.tanh(S / softcap)
                S = softcap * t
                e = e + 2.0**-22 * softcap
            bias = torch.zeros_like(S)
            if slopes is not None:
                bias = slopes[h].double() * (at[i][:, None] - col[None, :]).abs()
            e = e + 2.0**-22 * (S.abs() + bias)
            S = torch.where(see[i], S - bias, -math.inf)
            lse = torch.logsumexp(S, 1) if nk else torch.full((nq,), -math.inf, dtype=torch.float64, device=dev)
            P = torch.where(see[i], torch.exp(S - lse[:, None]), 0.0)
            # the bias of keys that carry no weight is large: only errors of weights that count are taken
            em = torch.where(P > 1e-12, e, 0.0).amax(1, keepdim=True) if nk else torch.zeros(nq, 1, dtype=torch.float64, device=dev)
            r["lse"][i, h] = lse
            r["e_lse"][i, h] = em[:, 0] + 2.0**-18 + 2.0**-22 * torch.where(lse.isinf(), 0.0, lse.abs())
            O = P @ V
            r["out"][i, :, h] = O
            E = u * O.abs() + (u + em + 2.0**-18) * (P @ V.abs()) + tiny * V.abs().sum(0) + 2 * tiny
            r["e_out"][i, :, h] = E
            if do is None:
                continue
            D = do[i, :, h].detach().double()
            D = torch.where(see[i].any(1)[:, None], D, 0.0)
            w = 2 * em + 2.0**-18 + torch.where(lse.isinf(), 0.0, lse.abs())[:, None] * 2.0**-22
            dP = D @ V.T
            delta = (D * O).sum(1, keepdim=True)
            dS = P * (dP - delta) * (1 - t * t)
            edS = (u + w) * dS.abs() + P * (g * (D.abs() @ V.abs().T) + (D.abs() * E).sum(1, keepdim=True))
            edS = edS + P * (2.0**-22 + 2 * w) * (dP.abs() + delta.abs())
            edS = edS + tiny * D.abs().max()  # dS is scaled by the largest |dO| before it is rounded
            r["dq"][i, :, h] = scale * dS @ K
            r["e_dq"][i, :, h] += abs(scale) * edS @ K.abs()
            r["dk"][i, :, kv] += scale * dS.T @ Q
            r["e_dk"][i, :, kv] += abs(scale) * edS.T @ Q.abs()
            r["dv"][i, :, kv] += P.T @ D
            r["e_dv"][i, :, kv] += ((u + w) * P + tiny).T @ D.abs()
    for n in ("dq", "dk", "dv"):
        r["e_" + n] += u * r[n].abs() + 2.0**-18 * r["e_" + n] + 2 * tiny + 1e-30
    r["e_out"] += 1e-30
    return r


def check(name, got, ref):
    """Fails where an element of ``got`` is further from the 64-bit value than its bound."""
    want, bound = ref[name], ref["e_" + name]
    got = got.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(got.isfinite(), want.isfinite()), f"{name}: not finite in other places"
    fin = want.isfinite()
    off = ((got - want).abs() - bound)[fin]
    if off.numel() and float(off.max()) > 0:
        at = int(((got - want).abs() - bound).nan_to_num(-1).argmax())
        raise AssertionError(f"{name}: {int((off > 0).sum())} of {off.numel()} elements are out of bounds, worst at {at}: "
                             f"{float(got.flatten()[at])} for {float(want.flatten()[at])}, bound {float(bound.flatten()[at]):.3g}")
