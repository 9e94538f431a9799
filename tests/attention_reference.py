"""Shared-prefix attention and the cache's quantisation in 64 bits, and how far the kernels may be from them."""
from __future__ import annotations

import math

import torch

FP8 = {"e4m3": (torch.float8_e4m3fn, 448.0, 3, -6), "e5m2": (torch.float8_e5m2, 57344.0, 2, -14)}
TYPES = ("f16", "int8", "e4m3", "e5m2")


def quantise(x: torch.Tensor, dtype: str):
    """(elements, FP32 scales or None) of FP16 vectors [..., D], each element from the exact quotient."""
    if dtype == "f16":
        return x.clone(), None
    wide = x.double()
    a = torch.where(torch.isfinite(wide), wide.abs(), 0.0).amax(-1)
    if dtype == "int8":
        scales = torch.where(a > 0, (a / 127.0).float(), torch.ones_like(a, dtype=torch.float32))
        q = torch.round(wide / scales.double()[..., None]).clamp(-127, 127)
        return torch.where(torch.isnan(q), 0.0, q).to(torch.int8), scales
    torch_type, largest, mantissa, least = FP8[dtype]
    exponent = torch.ceil(torch.log2(a.clamp_min(1e-30) / largest))
    exponent = torch.where(a > largest * torch.exp2(exponent), exponent + 1, exponent)
    exponent = torch.where(a <= largest * torch.exp2(exponent - 1), exponent - 1, exponent)
    scales = torch.where(a > 0, torch.exp2(exponent), torch.ones_like(a))
    y = wide / scales[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(1e-300))).clamp_min(least) - mantissa)
    q = (torch.round(y / step) * step).clamp(-largest, largest)
    return q.float().to(torch_type), scales.float()


def values_of(elements: torch.Tensor, scales):
    """What the elements stand for, in 64 bits."""
    return elements.double() if scales is None else elements.float().double() * scales.double()[..., None]


def attention(query, own, prefix, own_lengths=None, prefix_lengths=None, causal=False, scale=None):
    """(y, bound): query [B, L, H, D]; own and prefix are (k, v) [slots, tokens, heads, D] in 64 bits or None; lengths are lists.

    bound: how far an element of an FP16 result may be. With A = sum_j p_j |v_j|, n keys, and S the largest sum of
    |scale q_d k_d|, in units of the exact result:
      2^-11 |y|          the result's rounding to a half, and half its least step, 2^-25
      2^-11 A            each weight's rounding to a half
      n 2^-31 max|v|     weights below the least normal half: off by 2^-25, where a weight at the maximum is at least 2^6
      n 2^-23 A          sums of n products in 32 bits, each addition off by at most its last bit
      4 (D 2^-23 S) A    a score's own sum, off by D 2^-23 S, in a weight and in the weights' sum, doubled for the products with
                         the softmax scale and the key's scale
      2^-20 A            2^x and the division, a few last bits in 32
    """
    query = query.double()
    batch, tokens, heads, dim = query.shape
    scale = dim ** -0.5 if scale is None else scale
    y, bound = torch.zeros_like(query), torch.zeros_like(query)
    for b in range(batch):
        k, v, visible = [], [], []
        if prefix is not None:
            slot = b // (batch // prefix[0].shape[0])
            n = prefix[0].shape[1] if prefix_lengths is None else max(0, min(prefix_lengths[slot], prefix[0].shape[1]))
            k.append(prefix[0][slot, :n])
            v.append(prefix[1][slot, :n])
            visible.append(torch.ones((tokens, n), dtype=torch.bool, device=query.device))
        if own is not None:
            n = own[0].shape[1] if own_lengths is None else max(0, min(own_lengths[b], own[0].shape[1]))
            k.append(own[0][b, :n])
            v.append(own[1][b, :n])
            seen = torch.ones((tokens, n), dtype=torch.bool, device=query.device)
            if causal:
                seen = torch.arange(n, device=query.device)[None] <= n - tokens + torch.arange(tokens, device=query.device)[:, None]
            visible.append(seen)
        k, v, visible = torch.cat(k), torch.cat(v), torch.cat(visible, 1)
        repeat = heads // k.shape[1]
        for h in range(heads):
            kh, vh = k[:, h // repeat], v[:, h // repeat]
            s = (query[b, :, h] @ kh.t() * scale).masked_fill(~visible, -math.inf)
            top = s.amax(1, keepdim=True) if s.shape[1] else s.new_full((tokens, 1), -math.inf)
            w = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
            w = w.masked_fill(~visible, 0.0)
            total = w.sum(1, keepdim=True)
            p = w / torch.where(total > 0, total, 1.0)
            if torch.isfinite(vh).all():
                y[b, :, h] = p @ vh
            else:                                        # a hidden value takes no part, whatever it holds
                for i in range(tokens):
                    y[b, i, h] = p[i, visible[i]] @ vh[visible[i]]
            finite = torch.nan_to_num(vh, 0.0, 0.0, 0.0).abs()
            a = torch.nan_to_num(p) @ finite
            largest = (query[b, :, h].abs() @ torch.nan_to_num(kh, 0.0, 0.0, 0.0).abs().t()).amax() * abs(scale) if len(kh) else 0.0
            n = len(kh)
            bound[b, :, h] = 2 ** -11 * y[b, :, h].abs() + 2 ** -25 + (n * 2 ** -31 * finite.amax() if n else 0.0) + \
                a * (2 ** -11 + n * 2 ** -23 + 4 * dim * 2 ** -23 * largest + 2 ** -20)
    return y, bound


def off(got, want, bound):
    """The largest error in units of its bound; where the reference is not finite, got has to be so too."""
    got = got.double()
    odd = ~torch.isfinite(want)
    if odd.any() and torch.isfinite(got[odd]).any():
        return math.inf
    got, want, bound = got[~odd], want[~odd], bound[~odd]
    return float(((got - want).abs() / bound).amax().nan_to_num(math.inf)) if got.numel() else 0.0
