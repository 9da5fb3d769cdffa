"""The operators of long videos in float64, from their definitions: rotation by positions on several axes, attention in a window with first
keys that stay visible, attention states in blocks of 8 bits.  Test infrastructure; nothing here comes from the package."""
import math

import torch

PEAK = {"e4m3": 448.0, "int8": 127.0}


# ---- rotary positions ----------------------------------------------------------------------------------------------------------------

def pairs(dims, pairing, halves="axis"):
    """(a, b, axis, place in the axis) of every pair of elements."""
    D = sum(dims)
    axis = [(i, j) for i, d in enumerate(dims) for j in range(d // 2)]
    out, lo = [], 0
    if pairing == "rotate_half" and halves == "axis":
        for i, d in enumerate(dims):
            out += [(lo + j, lo + d // 2 + j, i, j) for j in range(d // 2)]
            lo += d
        return out
    for n, (i, j) in enumerate(axis):
        out.append((2 * n, 2 * n + 1, i, j) if pairing == "interleaved" else (n, n + D // 2, i, j))
    return out


def norm(x, kind, weight=None, bias=None, eps=1e-6):
    x = x.double()
    if kind is None:
        return x
    if kind == "layer_norm":
        x = x - x.mean(-1, keepdim=True)
    x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        x = x * weight.double()
    return x + bias.double() if kind == "layer_norm" and bias is not None else x


def rotate(x, positions, dims, base, pairing, halves="axis"):
    """x float64 ``[B,S,H,D]``, positions whole numbers ``[S,axes]`` or ``[B,S,axes]``."""
    y = x.clone()
    positions = positions.double()
    for a, b, i, j in pairs(dims, pairing, halves):
        angle = (positions[..., i] * float(base[i]) ** (-2.0 * j / dims[i])).unsqueeze(-1)
        c, s = angle.cos(), angle.sin()
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


# ---- attention in a window -------------------------------------------------------------------------------------------------------------

def visible(Sq, Sk, length, left, right, frame, sinks, q_begin):
    """bool ``[Sq, Sk]``: whole-number arithmetic, key by key."""
    p = (length - Sq if q_begin is None else q_begin) + torch.arange(Sq)[:, None]
    j = torch.arange(Sk)[None, :]
    mine, theirs = torch.div(p - sinks, frame, rounding_mode="floor"), torch.div(j - sinks, frame, rounding_mode="floor")
    seen = (j < length).expand(Sq, Sk)
    if right is not None:
        seen = seen & (theirs <= mine + right)
    if left is not None:
        seen = seen & ((theirs >= mine - left) | (j < sinks))
    return seen


def window_attention(q, k, v, left=None, right=None, frame=1, sinks=0, q_begin=None, kv_lens=None, scale=None):
    """(out, lse, sum of weights times |v|, largest sum |q_i k_i| scale) in float64; masked keys are not looked at.  Any device."""
    B, Sq, H, D = q.shape
    Sk, G = k.shape[1], H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(out)
    lse = torch.full((B, H, Sq), -math.inf, dtype=torch.float64, device=q.device)
    top = 0.0
    for b in range(B):
        n = Sk if kv_lens is None else min(max(int(kv_lens[b]), 0), Sk)
        seen = visible(Sq, Sk, n, left, right, frame, sinks, q_begin).to(q.device)
        used = seen.any(0).nonzero()[:, 0]
        if used.numel() == 0:
            continue
        hide = ~seen[:, used]
        for h in range(H):
            qh, kh, vh = q[b, :, h].double(), k[b, used, h // G].double(), v[b, used, h // G].double()
            s = (qh @ kh.T * scale).masked_fill(hide, -math.inf)
            l = torch.logsumexp(s, -1)
            w = torch.exp(s - torch.where(l > -math.inf, l, torch.zeros_like(l))[:, None])
            # (a weight of 0 leaves a value out, whatever it is)
            clean = torch.nan_to_num(vh, nan=0.0, posinf=0.0, neginf=0.0)
            o = w @ clean
            for j in ((vh != clean) | vh.isnan()).any(-1).nonzero()[:, 0].tolist():
                rows = ~hide[:, j]
                o[rows] += w[rows, j, None] * vh[j] - w[rows, j, None] * clean[j]
            out[b, :, h], lse[b, h], weight[b, :, h] = o, l, w @ clean.abs()
            top = max(top, float((qh.abs() @ torch.nan_to_num(kh).abs().T).max()) * scale)
    return out, lse, weight, top


# ---- states in blocks of 8 bits ------------------------------------------------------------------------------------------------------------

def quantize(x, fmt):
    """(elements as float64, exponents) of blocks of 32 along the last dimension: elements times 2^exponent are the values."""
    x = x.double().unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, -127.0)
    for n in range(-127, 128):                       # the smallest that holds
        e = torch.where((amax > PEAK[fmt] * 2.0 ** (n - 1)) & (n > -127), torch.full_like(e, float(n)), e)
    y = torch.ldexp(x, -e.int())
    if fmt == "int8":
        y = torch.round(y)
    else:
        step = torch.ldexp(torch.ones_like(y), torch.clamp(torch.frexp(y)[1] - 1, min=-6) - 3)
        y = torch.round(y / step) * step
    return y.flatten(-2), e.squeeze(-1)


def value(elements, exponents):
    return torch.ldexp(elements.double().unflatten(-1, (-1, 32)), exponents.int().unsqueeze(-1)).flatten(-2)


def merge(states):
    """states: (out, lse [B,H,S]) in any precision -> float64 (out, lse)."""
    lses = torch.stack([l.double() for _, l in states])
    total = torch.logsumexp(lses, 0)
    out = 0.0
    for (o, _), l in zip(states, lses):
        w = torch.where(l > -math.inf, torch.exp(l - torch.where(total > -math.inf, total, torch.zeros_like(total))), torch.zeros_like(l))
        w = w.transpose(1, 2).unsqueeze(-1)
        out = out + torch.where(w > 0, w * o.double(), torch.zeros_like(w))
    return out, total
