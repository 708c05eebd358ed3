"""CPU oracle, in 64 bits, of the operators around the log-prob path.  TEST INFRASTRUCTURE ONLY.

``norm_rope`` restates the reference's norm-and-rope kernel (mlx-impl/model.py:105-194: RMS norm of
each head, then the rotation of its two halves); ``attention`` the attention of the decode step
over a prompt's cache and a completion's (mlx-impl/model.py:428, node.py:529-555); ``policy_loss``
has no counterpart there (the loss belongs to the reference's external trainer).  Parity is by
formula; tests/test_step_oracle.py holds the gradients against differences.
"""
from __future__ import annotations

import torch


def _f64(x):
    return x.detach().cpu().double()


def rope(y, table, positions, back=False):
    """Heads ``[T, H, D]`` turned by their token's angles (or back)."""
    half = y.shape[-1] // 2
    rows = _f64(table)[positions.detach().cpu().long()]
    cos, sin = rows[:, None, :half], rows[:, None, half:]
    if back:
        sin = -sin
    a, b = y[..., :half], y[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def norm_rope(x, weight, table, positions, eps):
    """``(z, size)`` for heads ``x [T, H, D]``; ``size`` bounds what was added up for each element."""
    x, w = _f64(x), _f64(weight)
    y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    half = x.shape[-1] // 2
    rows = _f64(table)[positions.detach().cpu().long()].abs()
    cos, sin = rows[:, None, :half], rows[:, None, half:]
    a, b = y[..., :half].abs(), y[..., half:].abs()
    return rope(y, table, positions), torch.cat([a * cos + b * sin, b * cos + a * sin], dim=-1)


def norm_rope_backward(x, weight, grad, table, positions, eps):
    """``(dx, dw, size of dx, size of dw)``."""
    x, w = _f64(x), _f64(weight)
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    dy = rope(_f64(grad), table, positions, back=True)
    n, g = x * r, dy * w
    mean = (g * n).mean(-1, keepdim=True)
    size = r * (_f64(grad).abs().amax(-1, keepdim=True) * 2 * w.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    return r * (g - n * mean), (dy * n).sum((0, 1)), size, (dy * n).abs().sum((0, 1))


def pages(pool, table, length):
    """``[length, kv_heads, D]`` of one table's pages; entries outside the pool read as zeros."""
    num_blocks, kv, bs, d = pool.shape
    length = max(0, min(int(length), len(table) * bs))
    out = torch.zeros((length, kv, d), dtype=torch.float64)
    for i in range((length + bs - 1) // bs):
        page = int(table[i])
        n = min(bs, length - i * bs)
        if 0 <= page < num_blocks:
            out[i * bs:i * bs + n] = _f64(pool[page])[:, :n].transpose(0, 1)
    return out


def attention(q, k_pool, v_pool, prefix_tables, prefix_lens, group_starts, tables, lengths, scale):
    """``(out, lse, size, reach)``: ``size`` the softmax-weighted sum of |v| of each output, ``reach``
    the largest |scaled score| bound of each row (scale |q| |k|)."""
    n, h, d = q.shape
    kv = k_pool.shape[1]
    r = h // kv
    out = torch.zeros((n, h, d), dtype=torch.float64)
    lse = torch.full((n, h), -float("inf"), dtype=torch.float64)
    size, reach = torch.zeros_like(out), torch.zeros((n, h), dtype=torch.float64)
    starts = [] if group_starts is None else [int(s) for s in group_starts]
    for b in range(n):
        keys, values = pages(k_pool, tables[b], lengths[b]), pages(v_pool, tables[b], lengths[b])
        for g in range(len(starts) - 1):
            if starts[g] <= b < starts[g + 1]:
                keys = torch.cat([pages(k_pool, prefix_tables[g], prefix_lens[g]), keys])
                values = torch.cat([pages(v_pool, prefix_tables[g], prefix_lens[g]), values])
        if len(keys) == 0:
            continue
        x = _f64(q[b]).view(kv, r, d)
        s = torch.einsum("krd,tkd->krt", x, keys) * scale
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("krt,tkd->krd", p, values).reshape(h, d)
        size[b] = torch.einsum("krt,tkd->krd", p, values.abs()).reshape(h, d)
        lse[b] = torch.logsumexp(s, -1).reshape(h)
        reach[b] = (x.norm(dim=-1) * keys.norm(dim=-1).amax(0)[:, None] * scale).reshape(h)
    return out, lse, size, reach


def policy_loss(logits, ids, old, advantages, lengths, temp, starts=None, ref=None, clip_low=0.2,
                clip_high=0.2, kl_coef=0.0, reduction="token", grad_scale=1.0):
    """``(loss, logprobs, grad, slope)``; ``slope`` ``[n_seq, seq_len]`` is w (|a| rho + beta (1 + e^d))
    / T, what an error of the log-prob is multiplied with."""
    n, length, vocab = logits.shape
    lg, old = _f64(logits), _f64(old)
    adv = _f64(advantages)
    grad = torch.zeros_like(lg)
    lps, slopes = torch.zeros((n, length), dtype=torch.float64), torch.zeros((n, length), dtype=torch.float64)
    windows = []
    for i in range(n):
        st = 0 if starts is None else max(0, min(int(starts[i]), length))
        windows.append((st, st + max(0, min(int(lengths[i]), length - st))))
    total = sum(e - s for s, e in windows)
    loss = 0.0
    for i, (s, e) in enumerate(windows):
        if e == s:
            continue
        x = torch.log_softmax(lg[i, s:e] / temp, -1)
        t = ids[i, s:e].detach().cpu().long()[:, None]
        lp = x.gather(1, t)[:, 0]
        a = adv[i, s:e] if adv.dim() == 2 else adv[i]
        rho = (lp - old[i, s:e]).exp()
        kept = rho.clamp(1 - clip_low, 1 + clip_high)
        l = -torch.minimum(rho * a, kept * a)
        slope = torch.where(rho * a <= kept * a, -a * rho, torch.zeros_like(rho))
        reach = (a * rho).abs() * torch.ones_like(rho)
        if kl_coef:
            d = _f64(ref)[i, s:e] - lp
            l = l + kl_coef * (d.exp() - d - 1)
            slope = slope + kl_coef * (1 - d.exp())
            reach = reach + kl_coef * (1 + d.exp())
        w = 1.0 / total if reduction == "token" else 1.0 / (n * (e - s))
        loss = loss + (w * l).sum()
        g = slope * w * grad_scale / temp
        gr = -g[:, None] * x.exp()
        gr.scatter_add_(1, t, g[:, None])
        grad[i, s:e], lps[i, s:e], slopes[i, s:e] = gr, lp, reach * w * abs(grad_scale) / temp
    return torch.as_tensor(loss, dtype=torch.float64), lps, grad, slopes
