"""CPU tests: the 64-bit oracle of the operators around the log-prob path against autograd, against
differences and against algebra, and the refusals of their C entry points (made on the host, before
anything is launched)."""
import ctypes
import math

import pytest
import torch

from oracle import step


def _table(n, d, base=10000.0):
    half = d // 2
    angle = torch.arange(n, dtype=torch.float64)[:, None] * base ** (-torch.arange(half, dtype=torch.float64) / half)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def test_rotation_keeps_lengths_and_depends_on_distances_only():
    g = torch.Generator().manual_seed(3)
    x = torch.randn((2, 1, 16), generator=g, dtype=torch.float64)
    t = _table(200, 16)
    y = step.rope(x, t, torch.tensor([7, 31]))
    assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1), rtol=1e-6)
    z = step.rope(x, t, torch.tensor([107, 131]))
    assert abs(float((y[0] * y[1]).sum() - (z[0] * z[1]).sum())) < 1e-5
    assert torch.allclose(step.rope(y, t, torch.tensor([7, 31]), back=True), x, atol=1e-6)


def test_norm_rope_gradient_against_differences():
    g = torch.Generator().manual_seed(4)
    x = torch.randn((3, 2, 16), generator=g, dtype=torch.float64)
    w = 1 + 0.2 * torch.randn(16, generator=g, dtype=torch.float64)
    dz = torch.randn((3, 2, 16), generator=g, dtype=torch.float64)
    t, pos, eps = _table(50, 16), torch.tensor([0, 11, 49]), 1e-6
    dx, dw, _, _ = step.norm_rope_backward(x, w, dz, t, pos, eps)

    def f(x, w):
        return float((step.norm_rope(x, w, t, pos, eps)[0] * dz).sum())

    h = 1e-5
    for i in [(0, 0, 0), (1, 1, 7), (2, 0, 15)]:
        e = torch.zeros_like(x)
        e[i] = h
        assert abs((f(x + e, w) - f(x - e, w)) / (2 * h) - float(dx[i])) < 1e-8
    for i in (0, 9):
        e = torch.zeros_like(w)
        e[i] = h
        assert abs((f(x, w + e) - f(x, w - e)) / (2 * h) - float(dw[i])) < 1e-8


@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_loss_gradient_against_differences(reduction):
    g = torch.Generator().manual_seed(5)
    x = torch.randn((2, 3, 11), generator=g, dtype=torch.float64)
    ids = torch.randint(0, 11, (2, 3), generator=g)
    lp = torch.log_softmax(x / 0.8, -1).gather(-1, ids[..., None])[..., 0]
    old = lp + torch.tensor([[0.5, -0.05, -0.4], [0.1, -0.6, 0.3]])     # both sides of the clip
    ref, adv = lp + 0.3, torch.tensor([1.3, -0.7])
    kw = dict(ref=ref, kl_coef=0.1, clip_low=0.2, clip_high=0.3, reduction=reduction, grad_scale=2.0)
    lens, st = torch.tensor([2, 3]), torch.tensor([1, 0])
    loss, lps, grad, _ = step.policy_loss(x, ids, old, adv, lens, 0.8, st, **kw)
    assert float(lps[0, 0]) == 0 and float(grad[0, 0].abs().max()) == 0
    h = 1e-5
    for i in [(0, 1, 2), (0, 2, int(ids[0, 2])), (1, 0, 4), (1, 1, int(ids[1, 1])), (1, 2, 10), (0, 0, 3)]:
        e = torch.zeros_like(x)
        e[i] = h
        up = step.policy_loss(x + e, ids, old, adv, lens, 0.8, st, **kw)[0]
        down = step.policy_loss(x - e, ids, old, adv, lens, 0.8, st, **kw)[0]
        assert abs(float(up - down) / (2 * h) * 2.0 - float(grad[i])) < 1e-8
    assert math.isfinite(float(loss))


def test_attention_of_a_shared_prefix_is_attention_over_the_whole():
    g = torch.Generator().manual_seed(6)
    q = torch.randn((2, 4, 8), generator=g)
    k, v = torch.randn((6, 2, 4, 8), generator=g), torch.randn((6, 2, 4, 8), generator=g)
    out, lse, _, _ = step.attention(q, k, v, torch.tensor([[5, 1]]), [6], [0, 2],
                                    torch.tensor([[0, 2], [3, 4]]), [3, 8], 0.3)
    # the same tokens laid out in one table per sequence
    k2 = torch.zeros((2, 2, 16, 8))
    v2 = torch.zeros((2, 2, 16, 8))
    for b, (own, n) in enumerate((([0, 2], 3), ([3, 4], 8))):
        for dst, pool in ((k2, k), (v2, v)):
            rows = torch.cat([pool[5], pool[1][:, :2]], 1)
            tail = torch.cat([pool[own[0]], pool[own[1]]], 1)[:, :n]
            dst[b, :, :6 + n] = torch.cat([rows, tail], 1)
    out2, lse2, _, _ = step.attention(q, k2, v2, None, None, None, torch.tensor([[0], [1]]), [9, 14], 0.3)
    assert torch.allclose(out, out2) and torch.allclose(lse, lse2)


def test_norm_rope_refusals(built_lib):
    from tome_b200 import _lib
    lib, p, odd = _lib.lib, ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1008)

    def fwd(qkv=p, dtype=1, tokens=4, heads=2, kv=1, dim=64, stride=256, table=8, eps=1e-6, pos=p, q=p, k=p):
        return lib.tome_qk_norm_rope(qkv, dtype, tokens, heads, kv, dim, stride, p, p, p, table, pos, eps, q, k,
                                     None, None)
    assert fwd(dtype=3) == -3
    assert fwd(tokens=-1) == -4 and fwd(heads=0) == -4 and fwd(kv=0) == -4 and fwd(table=0) == -4
    assert fwd(dim=8) == -8 and fwd(dim=72) == -8 and fwd(dim=272) == -8
    assert fwd(stride=255) == -5 and fwd(stride=260) == -5
    assert fwd(eps=-1.0) == -4 and fwd(eps=float("nan")) == -4
    assert fwd(qkv=None) == -1 and fwd(pos=None) == -1 and fwd(q=odd) == -2
    assert fwd(tokens=0, qkv=None, q=None, k=None) == 0

    def app(n_seq=4, bs=16, blocks=4, num=8, seq_ids=None, tables=p, at=p, pool=p, tokens=4):
        return lib.tome_qk_norm_rope_append(p, 1, tokens, 2, 1, 64, 256, p, p, p, 8, p, 1e-6, seq_ids, tables, at,
                                            n_seq, bs, blocks, num, p, pool, p, None, None)
    assert app(n_seq=3) == -4 and app(bs=0) == -4 and app(blocks=-1) == -4 and app(num=-1) == -4
    assert app(tables=None) == -1 and app(at=None) == -1 and app(pool=None) == -1
    assert app(tokens=0, n_seq=0) == 0

    need = lib.tome_qk_norm_rope_backward_workspace_bytes(64)
    assert need >= 2 * 64 * 4 and lib.tome_qk_norm_rope_backward_workspace_bytes(0) == 0

    def bwd(gq=p, gv=None, ws=p, size=need, dw=p):
        return lib.tome_qk_norm_rope_backward(gq, p, gv, p, 1, 4, 2, 1, 64, 256, p, p, p, 8, p, 1e-6, p, dw, p, ws,
                                              size, None, None)
    assert bwd(gq=None) == -1 and bwd(dw=None) == -1 and bwd(gv=odd) == -2
    assert bwd(ws=None) == -6 and bwd(size=need - 1) == -6 and bwd(ws=odd) == -2


def test_attention_refusals(built_lib):
    from tome_b200 import _lib
    lib, p, odd = _lib.lib, ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1008)
    size = lib.tome_shared_prefix_attention_workspace_bytes
    need = size(8, 2, 4, 2, 64)
    assert need > 0 and size(0, 2, 4, 2, 64) == 0 and size(8, 2, 4, 3, 64) == 0 and size(8, 2, 4, 2, 96) == 0

    def att(q=p, dtype=1, n=8, heads=4, kv=2, dim=64, stride=256, pool=p, bs=16, num=8, pt=p, starts=p, groups=2,
            pb=4, bt=p, ln=p, mb=4, scale=0.1, out=p, ws=p, wsb=need):
        return lib.tome_shared_prefix_attention(q, dtype, n, heads, kv, dim, stride, pool, p, bs, num, pt, p, starts,
                                                groups, pb, bt, ln, mb, scale, out, None, ws, wsb, None, None)
    assert att(dtype=0) == -3 and att(dtype=7) == -3
    assert att(n=-1) == -4 and att(heads=3) == -4 and att(kv=0) == -4 and att(groups=-1) == -4
    assert att(n=5000) == -9 and att(groups=2000) == -9
    assert att(dim=96) == -8 and att(dim=256) == -8 and att(heads=258, kv=2) == -8
    assert att(bs=0) == -4 and att(mb=-1) == -4 and att(pb=-1) == -4
    assert att(scale=0.0) == -4 and att(scale=float("nan")) == -4 and att(scale=float("inf")) == -4
    assert att(stride=255) == -5 and att(stride=260) == -5
    assert att(q=None) == -1 and att(pool=None) == -1 and att(ln=None) == -1 and att(out=None) == -1
    assert att(bt=None) == -1 and att(pt=None) == -1 and att(starts=None) == -1
    assert att(q=odd) == -2 and att(ws=odd) == -2
    assert att(wsb=need - 1) == -6 and att(ws=None) == -6
    assert att(pb=2 ** 30, bs=64) == -9                     # more keys than 32 bits count
    assert att(n=0, q=None) == 0


def test_policy_loss_refusals(built_lib):
    from tome_b200 import _lib
    lib, p, odd = _lib.lib, ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1008)

    def loss(lg=p, dtype=1, n=3, length=5, vocab=64, ids=p, old=p, ref=p, adv=p, temp=1.0, low=0.2, high=0.2,
             beta=0.1, scale=1.0, out=p, lp=p, grad=p):
        return lib.tome_grpo_policy_loss(lg, dtype, n, length, vocab, ids, old, ref, adv, 0, p, None, temp, low, high,
                                         beta, 0, scale, out, lp, grad, None, None)
    assert loss(dtype=2) == -3 and loss(dtype=-1) == -3
    assert loss(n=-1) == -4 and loss(vocab=0) == -4 and loss(length=-2) == -4
    assert loss(temp=0.0) == -7 and loss(temp=float("nan")) == -7
    assert loss(low=-0.1) == -4 and loss(high=float("nan")) == -4 and loss(beta=-1.0) == -4
    assert loss(scale=float("inf")) == -4
    assert loss(out=None) == -1 and loss(lg=None) == -1 and loss(ids=None) == -1 and loss(old=None) == -1
    assert loss(adv=None) == -1 and loss(lp=None) == -1 and loss(ref=None) == -1
    assert loss(lg=odd) == -2 and loss(grad=odd) == -2


def test_cpu_tensors_are_refused(built_lib):
    import tome_b200 as tb
    x = torch.zeros((2, 4 * 64), dtype=torch.bfloat16)
    w, t, pos = x[0, :64], torch.zeros((4, 64)), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros((2, 1, 4, 64), dtype=torch.bfloat16)
    with pytest.raises(tb.TomeRuntimeError):
        tb.qk_norm_rope(x, w, w, t, pos, 2, 1)
    with pytest.raises(tb.TomeRuntimeError):
        tb.qk_norm_rope_backward(x.view(2, 4, 64), x.view(2, 4, 64), x, w, w, t, pos)
    with pytest.raises(tb.TomeRuntimeError):
        tb.qk_norm_rope_append(x, w, w, t, pos, pool, pool, pos[:, None], pos)
    with pytest.raises(tb.TomeRuntimeError):
        tb.shared_prefix_attention(x.view(2, 4, 64), pool, pool, None, None, None, pos[:, None], pos)
    with pytest.raises(tb.TomeRuntimeError):
        tb.grpo_policy_loss(x.view(1, 2, 256), pos[None], t[:1, :2], t[:1, 0], pos[:1])


def test_rope_table():
    import tome_b200 as tb
    t = tb.rope_table(100000, 16, 10000.0, device="cpu")
    assert t.shape == (100000, 16) and t.dtype == torch.float32
    assert abs(float(t[99999, 0]) - math.cos(99999.0)) < 1e-6          # far positions keep their angle
    assert abs(float(t[12345, 8 + 3]) - math.sin(12345.0 * 10000.0 ** (-3 / 8))) < 1e-6
    for bad in ((0, 16), (4, 0), (4, 15)):
        with pytest.raises(ValueError):
            tb.rope_table(*bad, device="cpu")
