"""GPU tests of the clipped policy loss and its gradient against the 64-bit oracle.

Tolerances.  A log-prob: the log-sum of V exponentials, each with an argument of at most |x|/T that is
rounded three times (2^-22), ex2 (2^-22) and a sum whose chains are at most V / 256 + 30 long in a
thread and over threads; its own magnitude, rounded three times: e = 2^-22 (|x|max / T + 2) + 2^-24 (V / 256
+ 30) + 2^-22 |lp|.  A gradient: half a step for the store, and relative 4 e for p, plus what an error e of the
log-prob does to the slope, times p (or 1 at the target)."""
import pytest
import torch

from oracle import step

pytestmark = pytest.mark.gpu


def _case(n, length, vocab, dtype, seed, temp=0.9, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (scale * torch.randn((n, length, vocab), generator=g)).to(dtype)
    ids = torch.randint(0, vocab, (n, length), generator=g, dtype=torch.int32)
    lp = torch.log_softmax(x.double() / temp, -1).gather(-1, ids.long()[..., None])[..., 0]
    drift = 0.3 * torch.randn((n, length), generator=g).double()
    # not within rounding of a clip border, where either side's slope is right
    for border in (0.2, 0.25):
        for b in (1 - border, 1 + border):
            drift = torch.where((drift.exp() - b).abs() < 1e-2, drift + 0.05, drift)
    return {"logits": x, "ids": ids, "old": (lp - drift).float(), "ref": (lp + 0.3 * torch.randn((n, length), generator=g)).float(),
            "adv": torch.randn(n, generator=g), "lengths": torch.randint(0, length + 1, (n,), generator=g, dtype=torch.int32),
            "temp": temp}


def _run(c, device, starts=None, kl=0.05, reduction="token", grad_scale=1.0, clip=(0.2, 0.25), **kw):
    import tome_b200
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    got = tome_b200.grpo_policy_loss(to(c["logits"]), to(c["ids"]), to(c["old"]), to(c["adv"]), to(c["lengths"]), c["temp"],
                                     starts=to(starts), ref_logprobs=to(c["ref"]), clip_low=clip[0], clip_high=clip[1],
                                     kl_coef=kl, reduction=reduction, grad_scale=grad_scale, check=True, **kw)
    loss, lp, grad, slope = step.policy_loss(c["logits"], c["ids"], c["old"], c["adv"], c["lengths"], c["temp"], starts,
                                             c["ref"], clip[0], clip[1], kl, reduction, grad_scale)
    T, vocab, dtype = c["temp"], c["logits"].shape[2], c["logits"].dtype
    x = c["logits"].double()
    xmax = x.masked_fill(~torch.isfinite(x), 0).abs().amax(-1) / T
    e = 2.0 ** -22 * (xmax + 2) + 2.0 ** -24 * (vocab / 256 + 30) + 2.0 ** -22 * lp.abs()
    assert bool(((got[1].cpu().double() - lp).abs() <= e).all())
    # the loss: every term moves by at most the slope times e, plus its own roundings
    terms = (slope * T / abs(grad_scale) * (e + 2.0 ** -20)).sum() if grad_scale else None
    assert got[0].dtype == torch.float32 and got[0].shape == ()
    if terms is not None:
        assert abs(float(got[0]) - float(loss)) <= float(terms) + 2.0 ** -23 * abs(float(loss)) + 1e-30
    if len(got) == 3:
        p = torch.softmax(x / T, -1)
        one = torch.zeros_like(p).scatter_(-1, c["ids"].long()[..., None], 1.0)
        u, f = torch.finfo(dtype).eps / 2, torch.finfo(dtype)
        tol = (u * grad.abs() + (p + one) * (slope * (6 * e + 2.0 ** -20))[..., None] + f.smallest_normal * f.eps
               + 2.0 ** -126 * (1 + slope[..., None]))
        off = (got[2].cpu().double() - grad).abs()
        assert bool((off <= tol).all()), float((off / tol).max())
        active = lp != 0
        assert not bool(got[2].cpu()[~active.bool()].any())
        return got, grad
    return got, None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 100, 1000, 4097, 12289, 50257, 151936])
def test_vocabularies(cuda_device, vocab, dtype):
    """Rows off the 16-byte grid, shorter than a vector, longer than a ring."""
    _run(_case(3, 5, vocab, dtype, vocab), cuda_device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,length,vocab", [(1, 1, 40000), (2, 1, 151936), (7, 40, 30000), (40, 20, 20001), (1, 900, 3001)])
def test_row_counts(cuda_device, n, length, vocab, dtype):
    """Each number of CTAs that share a row, rows fewer and more than the clusters."""
    c = _case(n, length, vocab, dtype, n + length)
    c["lengths"].fill_(length)
    _run(c, cuda_device)


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("kl", [0.0, 0.3])
def test_windows_reductions_and_coefficients(cuda_device, reduction, kl):
    c = _case(6, 12, 5000, torch.bfloat16, 3)
    c["lengths"] = torch.tensor([12, 0, 5, 100, -2, 3], dtype=torch.int32)
    starts = torch.tensor([0, 3, 4, 9, 2, 40], dtype=torch.int32)
    _run(c, cuda_device, starts, kl, reduction, grad_scale=3.0)
    _run(c, cuda_device, starts, kl, reduction, clip=(0.0, 0.0))
    _run(c, cuda_device, None, kl, reduction, clip=(1e9, 1e9))
    got, _ = _run(c, cuda_device, None, kl, reduction, grad_scale=0.0)
    assert not bool(got[2].any())
    _run(c, cuda_device, None, kl, reduction, return_grad=False)
    c["adv"] = torch.randn((6, 12), generator=torch.Generator().manual_seed(1))
    _run(c, cuda_device, starts, kl, reduction)


def test_masked_logits_and_magnitudes(cuda_device):
    """Masks of -inf and of the type's lowest value, a single live column, logits in the thousands."""
    for dtype in (torch.float32, torch.bfloat16):
        c = _case(4, 3, 3001, dtype, 7)
        x = c["logits"]
        keep = c["ids"].long()[..., None]
        kept = x.gather(-1, keep)
        x[0, :, ::2] = -float("inf")
        x[1, :, 5:] = torch.finfo(dtype).min
        x[2] = -float("inf")
        x.scatter_(-1, keep, kept)
        x[3] = x[3] * 300
        lp = torch.log_softmax(x.double() / c["temp"], -1).gather(-1, keep)[..., 0]
        c["old"], c["ref"] = (lp - 0.05).float(), (lp + 0.1).float()
        c["lengths"].fill_(3)
        got, _ = _run(c, cuda_device)
        assert float(got[1][2].abs().max()) == 0.0          # one live column: log-prob 0, no gradient
        assert float(got[2][2].abs().max()) == 0.0


def test_nan_and_bad_targets_stay_in_their_rows(cuda_device):
    import tome_b200
    c = _case(3, 4, 2000, torch.bfloat16, 8)
    c["lengths"].fill_(4)
    dev = {k: v.to(cuda_device) if isinstance(v, torch.Tensor) else v for k, v in c.items()}

    def call():
        return tome_b200.grpo_policy_loss(dev["logits"], dev["ids"], dev["old"], dev["adv"], dev["lengths"], c["temp"])
    want = call()
    dev["logits"][1, 2, 77] = float("nan")
    dev["ids"][2, 0], dev["ids"][0, 3] = 2000, -1
    loss, lp, grad = call()
    with pytest.raises(tome_b200.TomeRuntimeError, match="target"):
        tome_b200.check_device_status(cuda_device)
    bad = torch.zeros((3, 4), dtype=torch.bool, device=cuda_device)
    bad[1, 2] = bad[2, 0] = bad[0, 3] = True
    assert bool(loss.isnan()) and bool(lp[bad].isnan().all()) and bool(grad[bad].isnan().all())
    assert torch.equal(lp[~bad], want[1][~bad]) and torch.equal(grad[~bad], want[2][~bad])
    # outside a window neither is looked at
    dev["lengths"].zero_()
    loss, lp, grad = call()
    tome_b200.check_device_status(cuda_device)
    assert float(loss) == 0.0 and not bool(lp.any()) and not bool(grad.any())


def test_far_ratios(cuda_device):
    """A policy that moved far: the clip bounds one side, the other grows without turning NaN."""
    c = _case(2, 2, 500, torch.float32, 9)
    c["lengths"].fill_(2)
    lp = torch.log_softmax(c["logits"].double() / c["temp"], -1).gather(-1, c["ids"].long()[..., None])[..., 0]
    c["old"] = (lp - torch.tensor([[20.0, -20.0], [20.0, -20.0]])).float()
    c["adv"] = torch.tensor([1.0, -1.0])
    _run(c, cuda_device, kl=0.0)


def test_agrees_with_dual_scoring(cuda_device):
    """The same log-probs as grpo_dual_logprob_kl, whose KL is what the loss adds."""
    import tome_b200
    c = _case(4, 6, 30000, torch.bfloat16, 10, temp=0.7)
    g = torch.Generator().manual_seed(3)
    ref_logits = (c["logits"].float() + 0.1 * torch.randn(c["logits"].shape, generator=g)).to(torch.bfloat16)
    dev = [x.to(cuda_device) for x in (c["logits"], ref_logits, c["ids"], c["lengths"])]
    p, r, kl = tome_b200.grpo_dual_logprob_kl(*dev, 0.7)
    zero = torch.zeros(4, device=cuda_device)
    loss, lp = tome_b200.grpo_policy_loss(dev[0], dev[2], p, zero, dev[3], 0.7, ref_logprobs=r, kl_coef=1.0,
                                          return_grad=False)
    # the scoring kernel takes a quarter of its exponentials from a polynomial (7.5e-5)
    assert float((lp - p).abs().max()) <= 1e-4
    assert abs(float(loss) - float(kl.sum() / c["lengths"].sum())) <= 1e-4


def test_repetition_streams_graphs_and_out(cuda_device):
    import tome_b200
    c = _case(5, 9, 20001, torch.bfloat16, 11)
    dev = {k: v.to(cuda_device) if isinstance(v, torch.Tensor) else v for k, v in c.items()}

    def call(**kw):
        return tome_b200.grpo_policy_loss(dev["logits"], dev["ids"], dev["old"], dev["adv"], dev["lengths"], c["temp"],
                                          ref_logprobs=dev["ref"], kl_coef=0.1, **kw)
    want = call()
    out = torch.full_like(dev["logits"], 5.0)
    got = call(out_grad=out)
    assert got[2].data_ptr() == out.data_ptr()
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        other = call()
    side.synchronize()
    odd = torch.zeros(dev["logits"].numel() + 1, dtype=torch.bfloat16, device=cuda_device)
    odd[1:] = dev["logits"].reshape(-1)
    keep, dev["logits"] = dev["logits"], odd[1:].view(dev["logits"].shape)   # off the grid: copied
    moved = call()
    dev["logits"] = keep.transpose(0, 1).contiguous().transpose(0, 1)          # not contiguous: copied
    turned = call()
    dev["logits"] = keep
    for g in (got, other, moved, turned):
        assert all(torch.equal(a, b) for a, b in zip(want, g))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    dev["lengths"].copy_(torch.tensor([9, 1, 0, 4, 9], dtype=torch.int32))
    dev["logits"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(call(), held))
    for kw in ({"out_grad": dev["logits"]}, {"out_grad": out.float()}, {"out_grad": out[:1]}, {"reduction": "sum"},
               {"out_grad": out, "return_grad": False}, {"clip_low": -1.0}, {"grad_scale": float("nan")}):
        with pytest.raises((ValueError, TypeError)):
            call(**kw)
    with pytest.raises(ValueError):
        tome_b200.grpo_policy_loss(dev["logits"], dev["ids"], dev["old"], dev["adv"], dev["lengths"], kl_coef=0.1)
    with pytest.raises(ValueError):
        tome_b200.grpo_policy_loss(dev["logits"], dev["ids"], dev["old"].t(), dev["adv"], dev["lengths"])
    with pytest.raises(TypeError):
        tome_b200.grpo_policy_loss(dev["logits"].half(), dev["ids"], dev["old"], dev["adv"], dev["lengths"])
    empty = tome_b200.grpo_policy_loss(dev["logits"][:0], dev["ids"][:0], dev["old"][:0], dev["adv"][:0],
                                       dev["lengths"][:0])
    assert float(empty[0]) == 0.0 and empty[2].shape == (0, 9, 20001)


def test_gradient_continues_through_autograd(cuda_device):
    """The gradient handed to logits.backward is that of autograd through the same formula."""
    import tome_b200
    g = torch.Generator().manual_seed(12)
    hidden = torch.randn((2, 3, 16), generator=g).to(cuda_device)
    w = torch.randn((500, 16), generator=g).to(cuda_device).requires_grad_()
    ids = torch.randint(0, 500, (2, 3), generator=g, dtype=torch.int32).to(cuda_device)
    old = torch.full((2, 3), -6.0, device=cuda_device)
    adv = torch.tensor([0.5, -1.0], device=cuda_device)
    lens = torch.tensor([3, 2], dtype=torch.int32, device=cuda_device)
    logits = hidden @ w.t()
    _, _, grad = tome_b200.grpo_policy_loss(logits, ids, old, adv, lens, clip_low=1e9, clip_high=1e9)
    logits.backward(grad)
    got, w.grad = w.grad, None
    lp = torch.log_softmax((hidden @ w.t()).double(), -1).gather(-1, ids.long()[..., None])[..., 0]
    mask = torch.arange(3, device=cuda_device) < lens[:, None]
    (-((lp - old).exp() * adv[:, None]) * mask).sum().div(5).backward()
    # two fp32 products of 16 and 6 terms, and the loss's own fp32 gradient
    assert float((got - w.grad).abs().max()) <= 2.0 ** -14 * float(w.grad.abs().max())


@pytest.mark.parametrize("n", [1023, 1024, 1025, 2500])
def test_many_sequences(cuda_device, n):
    """Many short sequences, most of them with rows outside their windows."""
    c = _case(n, 3, 300, torch.bfloat16, 13)
    starts = torch.randint(0, 4, (n,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    _run(c, cuda_device, starts)
    _run(c, cuda_device, None, reduction="sequence", return_grad=False)


@pytest.mark.parametrize("seed", range(4))
def test_ratio_keeps_its_bits(cuda_device, seed):
    """fp32 gradients of rows with two large logits; the others' exponentials (below e^-1000) add nothing,
    exactly.  So the sum s is off by an ex2 (2^-22) and three roundings, which reach the gradient twice,
    by log s in the ratio and by the division; log s itself by half a step of a number below 1 (2^-25);
    expf and the second ex2 by 2^-22 each; the exponent's one rounding, slope, weight and products by nine
    roundings: 2 (2^-22 + 3 2^-24) + 2^-25 + 2 2^-22 + 9 2^-24 < 2^-19, relative to slope times p (or
    times 1 at the target, where 1 - p may cancel).  (Roundings at the size of the logits, 2000 after
    the division, would be 2^-14 each.)"""
    import tome_b200
    n, length, vocab, T = 2, 8, 5000, 0.5
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn((n, length, vocab), generator=g)
    ids = torch.randint(0, vocab, (n, length), generator=g, dtype=torch.int32)
    ids.clamp_(min=1)
    x.scatter_(-1, ids.long()[..., None], 1000.0)                    # the target stands out, far from 0
    x[..., 0] = 1000.25
    lp = torch.log_softmax(x.double() / T, -1).gather(-1, ids.long()[..., None])[..., 0]
    old = (lp - 0.05 * torch.randn((n, length), generator=g).double()).float()
    adv, lengths = torch.tensor([1.0, -1.0]), torch.full((n,), length, dtype=torch.int32)
    _, _, grad = tome_b200.grpo_policy_loss(*(t.to(cuda_device) for t in (x, ids, old, adv, lengths)), T, check=True)
    want = step.policy_loss(x, ids, old, adv, lengths, T)[2]
    slope = want.gather(-1, ids.long()[..., None]).abs() / (1 - lp.exp())[..., None]
    one = torch.zeros_like(want).scatter_(-1, ids.long()[..., None], 1.0)
    p = torch.softmax(x.double() / T, -1)
    rel = 2.0 ** -19
    away = (x.double().amax(-1, keepdim=True) - x.double()) / T      # the exponent's size, rounded twice
    tol = slope * (p + one) * (rel + 2.0 ** -22 * away) + 2.0 ** -126
    off = (grad.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
