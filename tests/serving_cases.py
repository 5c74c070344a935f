"""The serving operators in 64 bits, as their definitions say, and how far kernels may be off."""
import math

import torch


def half_step(dtype) -> float:
    """What a rounding to `dtype` is off by at most, relative to the value."""
    return torch.finfo(dtype).eps / 2


def rotate(x, position, freqs, amp, interleaved):
    """x (heads, D) at a position, and a bound on what 32-bit arithmetic on 32-bit cosines is off by: cos and sin are off by 2^-22 (the
    angle, at most pi, is rounded once to 32 bits, 2^-23, and sincosf is off by an ulp or two), products and sum by 3 * 2^-24."""
    x, slack = x.double(), torch.zeros_like(x, dtype=torch.float64)
    if freqs is None:
        return x, slack
    half = freqs.numel()
    y = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = position * float(freqs[i])
        c, s = math.cos(angle) * amp, math.sin(angle) * amp
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
        slack[:, a] = slack[:, b] = (x[:, a].abs() + x[:, b].abs()) * abs(amp) * (2 ** -22 + 3 * 2 ** -24)
    return y, slack


def attend(q, k, v, scale, weight_step=0.0):
    """q (R, D) over k, v (n, D): (R, D) and a bound on the error in 32 bits before the last rounding. With A = sum of weights times |v|:
    a score of D products is off by scale * sum |q k| * (D + 2) * 2^-24, which moves weights and their sum (twice) by as much; the
    exponential adds 2^-21 for its argument of up to 16 or so and itself, the sums n * 2^-24, and weights rounded to a shorter type
    weight_step each."""
    q, k, v = q.double(), k.double(), v.double()
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    n, D = k.shape
    p = torch.softmax(q @ k.t() * scale, 1)
    off = abs(scale) * (q.abs() @ k.abs().t()).amax(1, keepdim=True) * (D + 2) * 2.0 ** -24
    return p @ v, (p @ v.abs()) * (2 * off + 2.0 ** -20 + n * 2.0 ** -24 + weight_step)


def within(got, want, slack, dtype):
    """Every entry within its slack and one rounding; an entry that is not finite has to be so in both."""
    if got.numel() == 0:
        return True, ""
    got, limit = got.double(), slack + (want.abs() + slack) * half_step(dtype) + torch.finfo(dtype).smallest_normal * 2.0 ** -9
    ok = (got - want).abs() <= limit
    return bool(ok.all()), f"worst {float(((got - want).abs() / limit).nan_to_num(9e9).max()):.2f} of what is allowed"


def sample(row, u, temperature, top_k, top_p, min_p) -> int:
    """One token from one row of logits (a 1-D tensor on the CPU)."""
    entries = [(-x, i) for i, x in enumerate(row.double().tolist()) if x == x and x != -math.inf]
    if not entries:
        return -1
    entries.sort()
    if temperature <= 0 or top_k == 1:
        return entries[0][1]
    if top_k > 0:
        entries = entries[:top_k]
    top = entries[0][0]
    ranked = [(math.exp((top - x) / temperature), i) for x, i in entries]
    if top_p < 1:
        mass, before, kept = top_p * math.fsum(w for w, _ in ranked), 0.0, []
        for w, i in ranked:
            if kept and before >= mass:
                break
            kept.append((w, i))
            before += w
        ranked = kept
    ranked = sorted((i, w) for w, i in ranked if w >= min_p)
    total, run = math.fsum(w for _, w in ranked), 0.0
    for i, w in ranked:
        run += w
        if run > u * total:
            return i
    return ranked[-1][0]
