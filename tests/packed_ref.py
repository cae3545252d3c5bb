"""Plain 64-bit forms of the operators over packed sets (attention, rope, group_norm), with the
error each may have: half a step of every rounding that the operator makes, counted through its
formula."""
import math

import torch

#: Half a step relative to the value: what one rounding to the type may be off by.
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}


def offsets(lengths, first=0):
    off = [first]
    for n in lengths:
        off.append(off[-1] + n)
    return off


def table(off, device="cuda"):
    return torch.tensor(off, dtype=torch.int32, device=device)


def attention(q, k, v, qo, ko, causal, scale):
    """(out, lse, weight) in 64 bits on q's device: weight[i, h, d] = sum_j p_j |v_j| / sum_j p_j, by
    which relative errors of the p_j reach the output, and reach = the largest sum of |q||k| scale."""
    nq, h, d = q.shape
    g = h // k.shape[1]
    out = torch.full((nq, h, d), math.nan, dtype=torch.float64, device=q.device)
    wgt = torch.zeros_like(out)
    lse = torch.full((nq, h), math.nan, dtype=torch.float64, device=q.device)
    reach = 0.0
    for s in range(len(qo) - 1):
        a, b, c, e = qo[s], qo[s + 1], ko[s], ko[s + 1]
        if a == b:
            continue
        if c == e:
            out[a:b], lse[a:b] = 0.0, -math.inf
            continue
        qs = q[a:b].double().transpose(0, 1)
        ks = k[c:e].double().repeat_interleave(g, 1).transpose(0, 1)
        vs = v[c:e].double().repeat_interleave(g, 1).transpose(0, 1)
        x = qs @ ks.transpose(1, 2) * scale
        reach = max(reach, float((qs.abs() @ ks.abs().transpose(1, 2)).max()) * scale)
        if causal:
            i = torch.arange(b - a, device=q.device)[:, None] + (e - c) - (b - a)
            x = x.masked_fill(torch.arange(e - c, device=q.device)[None] > i, -math.inf)
        m = x.amax(-1, keepdim=True).clamp_min(-1e300)
        p = torch.exp(x - m)
        l = p.sum(-1, keepdim=True)
        o = torch.where(l > 0, p @ vs / l, 0.0)
        w = torch.where(l > 0, p @ vs.abs() / l, 0.0)
        out[a:b], wgt[a:b] = o.transpose(0, 1), w.transpose(0, 1)
        lse[a:b] = (m + torch.log(l))[..., 0].transpose(0, 1)
    return out, lse, wgt, reach


def attention_tolerance(ref, wgt, reach, d, nk, dtype, out_dtype):
    """Per element. The output is rounded once (HALF of its type). Each p_j may be off by a share
    `rel`, which reaches the output times weight, once for the p_j and once for their sum:
    * 16-bit operands: p_j rounded to the type, HALF; its exponential is allowed 2^-13;
    * a score is a sum of d products in 32 bits and a product with the scale: at most (d + 3) half
      steps of the sum of its terms' magnitudes (reach); an error e of a score is a share e of p_j;
    * the sums over nk keys in 32 bits: at most nk half steps, in pieces of 64 keys or more that are
      added up one by one: 64 + nk / 64."""
    f = HALF[torch.float32]
    sums = (64 + nk / 64) * f
    rel = (d + 3) * f * reach + sums + (HALF[dtype] + 2 ** -13 if dtype != torch.float32 else 4 * f)
    return HALF[out_dtype] * ref.abs() * (1 + rel) + 2 * rel * wgt + 1e-30


def close(got, ref, tol):
    """Largest |got - ref| / tol over elements of `ref` that are numbers (NaN: not written)."""
    want = ~torch.isnan(ref)
    return float(((got.double() - ref).abs() / tol)[want].max()) if want.any() else 0.0


def rope(x, pos, sections, theta, layout, joint, inverse):
    n, h, d = x.shape
    half = d // 2
    out = x.double().clone()
    pair = 0
    for axis, size in enumerate(sections):
        for j in range(size):
            f = theta ** -((pair / half) if joint else (j / size))
            t = pos[:, axis].double() * f
            c, s = torch.cos(t)[:, None], torch.sin(t)[:, None] * (-1 if inverse else 1)
            ia, ib = (2 * pair, 2 * pair + 1) if layout == "pairs" else (pair, pair + half)
            a, b = x[..., ia].double(), x[..., ib].double()
            out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
            pair += 1
    return out


def group_norm(x, groups, w, b, off, eps, act):
    n, c = x.shape
    out = torch.full((n, c), math.nan, dtype=torch.float64, device=x.device)
    for s in range(len(off) - 1):
        a, e = off[s], off[s + 1]
        if a == e:
            continue
        y = x[a:e].double().view(e - a, groups, -1)
        mean = y.mean((0, 2), keepdim=True)
        y = (y - mean) / torch.sqrt(((y - mean) ** 2).mean((0, 2), keepdim=True) + eps)
        y = y.reshape(e - a, c)
        if w is not None:
            y = y * w.double()
        if b is not None:
            y = y + b.double()
        out[a:e] = y / (1 + torch.exp(-y)) if act == "silu" else y
    return out
