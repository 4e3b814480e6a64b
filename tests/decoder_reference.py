"""Plain fp64 forms of the decoder-layer operators, and the error bounds their kernels are held to."""
import math

import torch


def norm_quant(h, r, w, eps, group):
    """(y / scale unrounded, scales, s unrounded) in fp64 for [rows, cols] operands."""
    s = h.double() + r.double()
    y = s / (s.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    x, scales = torch.empty_like(y), []
    for c in range(0, y.shape[1], group or y.shape[1]):
        part = y[:, c : c + (group or y.shape[1])]
        largest = part.abs().amax(-1, keepdim=True)
        unit = torch.where(largest == 0, torch.ones_like(largest), largest / 448)
        x[:, c : c + part.shape[1]] = part / unit
        scales.append(unit)
    return x, torch.cat(scales, 1), s


def rotary(x, positions, inv_freq, sections, interleaved, inverse):
    """[B, S, N, D] turned in fp64; positions [A, B, S]."""
    angle = torch.cat([positions[a].double().unsqueeze(-1) * f.double()
                       for a, f in enumerate(torch.split(inv_freq, sections))], -1).unsqueeze(2)
    cos, sin = angle.cos(), angle.sin() * (-1 if inverse else 1)
    pairs = inv_freq.numel()
    y = x.double().clone()
    if interleaved:
        a, b = y[..., 0 : 2 * pairs : 2].clone(), y[..., 1 : 2 * pairs : 2].clone()
        y[..., 0 : 2 * pairs : 2], y[..., 1 : 2 * pairs : 2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = y[..., :pairs].clone(), y[..., pairs : 2 * pairs].clone()
        y[..., :pairs], y[..., pairs : 2 * pairs] = a * cos - b * sin, b * cos + a * sin
    return y


def visible(first, queries, keys, window, sinks, length):
    """[queries, keys] bool: query i sits at position first + i; positions from `length` on do not exist."""
    at = torch.arange(first, first + queries).unsqueeze(1)
    key = torch.arange(keys).unsqueeze(0)
    return (key <= at) & ((at - key < window) | (key < sinks)) & (at < length)


def attention(q, k, v, scale, window, sinks, lengths=None, dout=None):
    """fp64 attention of [B, N, Sq, D] queries, the last Sq of Sk positions.  Returns a dict: out, lse, `weight`
    (sum of p |v|, what the rounding of the probabilities acts on), and with dout the gradients."""
    B, N, Sq, D = q.shape
    Nk, Sk = k.shape[1:3]
    G = N // Nk
    q, k, v = q.double(), k.double(), v.double()
    out, weight = torch.zeros(B, N, Sq, D, dtype=torch.float64), torch.zeros(B, N, Sq, D, dtype=torch.float64)
    lse = torch.full((B, N, Sq), -math.inf, dtype=torch.float64)
    grads = {}
    if dout is not None:
        dout = dout.double()
        for name, like in (("dq", q), ("dk", k), ("dv", v)):
            grads[name] = torch.zeros_like(like, memory_format=torch.contiguous_format)
            grads[name + "_weight"] = torch.zeros_like(grads[name])
    for b in range(B):
        length = Sk if lengths is None else int(lengths[b])
        see = visible(Sk - Sq, Sq, Sk, window, sinks, length)
        rows = see.any(-1)
        for h in range(N):
            kk, vv = k[b, h // G].clone(), v[b, h // G].clone()
            kk[length:], vv[length:] = 0, 0
            qq = torch.where(rows.unsqueeze(1), q[b, h], torch.zeros_like(q[b, h]))
            s = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
            z = torch.logsumexp(s, -1)
            p = torch.where(see, (s - torch.where(rows, z, torch.zeros_like(z)).unsqueeze(1)).exp(), torch.zeros_like(s))
            out[b, h], weight[b, h], lse[b, h] = p @ vv, p @ vv.abs(), z
            if dout is not None:
                g = torch.where(rows.unsqueeze(1), dout[b, h], torch.zeros_like(dout[b, h]))
                slope = g @ vv.T
                delta = (g * out[b, h]).sum(-1, keepdim=True)
                ds = p * (slope - delta)
                # what the kernels round: P (dV) and dS (dQ, dK) to the operand type, and O inside delta, which holds
                # two roundings itself: the probabilities' and its own
                ds_size = p * (slope.abs() + delta.abs() + 2 * (g.abs() * weight[b, h]).sum(-1, keepdim=True))
                grads["dv"][b, h // G] += p.T @ g
                grads["dv_weight"][b, h // G] += p.T @ g.abs()
                grads["dq"][b, h] = ds @ kk * scale
                grads["dq_weight"][b, h] = ds_size @ kk.abs() * scale
                grads["dk"][b, h // G] += ds.T @ qq * scale
                grads["dk_weight"][b, h // G] += ds_size.T @ qq.abs() * scale
    return {"out": out, "lse": lse, "weight": weight, **grads}


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def attention_bound(want, weight, dtype):
    """Error bound of an attention result.  The stored value is rounded once (half a step of it).  Every term of the
    sum carries one rounding of its probability (or dS) to the operand type, half a step of the sum of the terms'
    sizes `weight`; and the error of its score in fp32: at most (D + 2) 2^-24 sum |q k| scale, for normal operands
    of D <= 128 below 130 * 6e-8 * 8 = 6.2e-5, twice (the term and the normalising sum), rounded up to 2e-4.
    fp16 probabilities below its smallest normal number are off by up to 2^-25 of the largest, which 1e-5 covers."""
    h = half_step(dtype)
    return want.abs() * h + weight * (h + 2e-4) + 1e-5


def fp16_gradient_bounds(q, k, v, scale, window, sinks, dout):
    """(gradients, bounds, spreads) of fp16 operands of any size, for one sequence and scores of normal size.  The spreads are
    standard deviations of dq and dk when every rounding is an independent error, evenly spread over half a step up and
    down (its square mean a third of the half step's square).

    Beside what attention_bound counts (each term's rounding, the scores' errors of 2e-4) fp16 has an end of its normal
    numbers, 2^-14, where a rounding is off by up to 2^-25 absolutely:
      of the result                2^-25
      of P 2^14 (dV)               2^-39 a pair
      of dS 2^s (dK), by the key   s brings B = max |dO| sum |V| + max |D| to 2^14 or more: 2^-25 B 2^-14 a pair
      of dS 2^s (dQ), by the row   s brings max |dO| to 2^7 or more: 2^-25 max |dO| 2^-7 a pair; where that would pass 65504,
                                   s brings 2 D max |dO| max |V| to 2^14 or more: 2^-25 of that 2^-14 a pair
      of out and its remainder in D: P times 2^-24 sum |dO| a pair."""
    _, N, Sq, D = q.shape
    Nk, Sk = k.shape[1:3]
    G = N // Nk
    h = half_step(torch.float16)
    q, k, v, g = (t[0].double() for t in (q, k, v, dout))
    see = visible(Sk - Sq, Sq, Sk, window, sinks, Sk)
    out = {x: torch.zeros_like(t) for x, t in (("dq", q), ("dk", k), ("dv", v))}
    bound = {x: torch.zeros_like(t) for x, t in out.items()}
    square = {x: torch.zeros_like(t) for x, t in out.items()}
    for n in range(N):
        j = n // G
        s = (q[n] @ k[j].T * scale).masked_fill(~see, -math.inf)
        # the forward's probabilities, relative to the largest, are normal numbers
        assert (s.amax(-1, keepdim=True) - s)[see].max() < 9.7
        p = s.softmax(-1)
        dp = g[n] @ v[j].T
        delta = (g[n] * (p @ v[j])).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        size = p * (dp.abs() + delta.abs() + 2 * (g[n].abs() * (p @ v[j].abs())).sum(-1, keepdim=True))
        most = g[n].abs().amax(-1, keepdim=True)
        lost_d = p * 2.0**-24 * g[n].abs().sum(-1, keepdim=True)
        over = 2.0**8 * (dp - delta).abs().amax(-1, keepdim=True) * p.amax(-1, keepdim=True) > 32768 * most
        least_q = torch.where(over, torch.maximum(2.0**-32 * most, 2.0**-39 * 2 * D * most * v[j].abs().max()), 2.0**-32 * most)
        b = g[j * G : j * G + G].abs().max() * v[j].abs().sum(-1) + max(
            (g[m] * ((q[m] @ k[j].T * scale).masked_fill(~see, -math.inf).softmax(-1) @ v[j])).sum(-1).abs().max() for m in range(j * G, j * G + G))
        out["dq"][n] = ds @ k[j] * scale
        bound["dq"][n] = (size * (h + 2e-4) + lost_d + see * least_q) @ k[j].abs() * scale
        out["dk"][j] += ds.T @ q[n] * scale
        bound["dk"][j] += (size * (h + 2e-4) + lost_d + see * (2.0**-39 * b)).T @ q[n].abs() * scale
        least_k = see * (2.0**-39 * b)
        square["dq"][n] = ((ds * h).square() + (see * least_q).square()) @ k[j].square() * scale**2 / 3
        square["dk"][j] += ((ds * h).square() + least_k.square()).T @ q[n].square() * scale**2 / 3
        out["dv"][j] += p.T @ g[n]
        bound["dv"][j] += (p * (h + 2e-4) + see * 2.0**-39).T @ g[n].abs()
    spread = {x: (square[x] + (t.half().double() - t).square()).sqrt().unsqueeze(0) for x, t in out.items() if x != "dv"}
    return {x: t.unsqueeze(0) for x, t in out.items()}, {x: (t + out[x].abs() * h + 2.0**-25).unsqueeze(0) for x, t in bound.items()}, spread


def wide_attention(q, k, v, scale, window, sinks, lengths, dout, dtype):
    """(results, bounds) of attention and its gradients for scores of any size.

    As attention_bound, with the errors of scores by their size: a score is off by (D + 2) 2^-24 sum |q k| scale, and where
    the row's lse is what a sum starts from by as much of |lse|; E is twice that, for the term and for the sum it is
    divided by.  fp16 adds the ends of its normal numbers: 2^-25 a probability of the forward, which are relative to a
    value of at least 1, and what fp16_gradient_bounds lists."""
    B, N, Sq, D = q.shape
    Nk, Sk = k.shape[1:3]
    G = N // Nk
    h, tiny = half_step(dtype), (1.0 if dtype == torch.float16 else 0.0)
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    out = {x: torch.zeros_like(t, memory_format=torch.contiguous_format) for x, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    out["lse"] = torch.full((B, N, Sq), -math.inf, dtype=torch.float64)
    bound = {x: torch.zeros_like(t) for x, t in out.items()}
    for b in range(B):
        see = visible(Sk - Sq, Sq, Sk, window, sinks, Sk if lengths is None else lengths[b])
        rows = see.any(-1, keepdim=True)
        for n in range(N):
            j = n // G
            qq, g = q[b, n] * rows, dout[b, n] * rows
            s = (qq @ k[b, j].T * scale).masked_fill(~see, -math.inf)
            z = torch.logsumexp(s, -1, keepdim=True)
            zz = torch.where(rows, z, torch.zeros_like(z))
            p = torch.where(see, (s - zz).exp(), torch.zeros_like(s))
            e = 2 * (D + 2) * 2.0**-24 * ((qq.abs() @ k[b, j].abs().T * scale * see).amax(-1, keepdim=True) + zz.abs())
            o, weight = p @ v[b, j], p @ v[b, j].abs()
            floor = tiny * 2.0**-25 * (see.double() @ v[b, j].abs())
            out["out"][b, n], out["lse"][b, n] = o, z[:, 0]
            bound["out"][b, n] = o.abs() * h + weight * (h + e) + floor + 2.0**-25
            bound["lse"][b, n] = (e + 2.0**-22 * zz.abs() + 2.0**-20)[:, 0]
            dp = g @ v[b, j].T
            delta = (g * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            size = p * (dp.abs() + delta.abs() + 2 * (g.abs() * weight).sum(-1, keepdim=True))
            lost_d = p * (g.abs() * (floor + 2.0**-24)).sum(-1, keepdim=True)
            most, all_v = g.abs().amax(-1, keepdim=True), v[b, j].abs()
            least_q = tiny * 2.0**-39 * 2 * D * most * all_v.max()  # of the two the larger
            least_k = tiny * 2.0**-39 * (dout[b].abs().max() * all_v.sum(-1) + dout[b].abs().max() * all_v.sum(-1).max())
            err_ds = size * (h + e) + lost_d
            out["dq"][b, n], out["dv"][b, j], out["dk"][b, j] = ds @ k[b, j] * scale, out["dv"][b, j] + p.T @ g, out["dk"][b, j] + ds.T @ qq * scale
            bound["dq"][b, n] = (err_ds + see * torch.maximum(least_q, 2.0**-32 * tiny * most)) @ k[b, j].abs() * scale
            bound["dk"][b, j] += (err_ds + see * least_k).T @ qq.abs() * scale
            bound["dv"][b, j] += (p * (h + e) + see * tiny * 2.0**-39).T @ g.abs()
    for x in ("dq", "dk", "dv"):
        bound[x] += out[x].abs() * h + 2.0**-25
    return out, bound
