"""GPU test of the operators as a rollout and a training step use them together: prompts are appended
to the paged cache once per group, completions are decoded over the shared pages, their tokens
are sampled and scored, and the policy loss and the norm's gradient follow.  Tolerances are those of
the operators' own tests; what goes through the same arithmetic twice has to agree to the bit."""
import pytest
import torch

from oracle import step

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, BLOCK = 8, 2, 64, 16
GROUPS, EACH = 2, 3
PREFIX = (21, 0)           # the second group has no prompt
STEPS, VOCAB, TEMP, EPS = 5, 1001, 0.8, 1e-6


def _model(device, dtype):
    g = torch.Generator().manual_seed(5)
    n = GROUPS * EACH
    width = (HEADS + 2 * KV) * DIM
    most_p, most_s = 2, 1
    pages = torch.randperm(GROUPS * most_p + n * most_s + 2, generator=g).to(torch.int32)
    rand = lambda *s: torch.randn(s, generator=g).to(dtype).to(device)  # noqa: E731
    return {
        "prompt": rand(sum(PREFIX), width), "tokens": rand(STEPS, n, width), "head": 0.1 * rand(HEADS * DIM, VOCAB),
        "qw": 1 + 0.1 * rand(DIM), "kw": 1 + 0.1 * rand(DIM),
        "k_pool": torch.zeros((len(pages), KV, BLOCK, DIM), dtype=dtype, device=device),
        "v_pool": torch.zeros((len(pages), KV, BLOCK, DIM), dtype=dtype, device=device),
        "prefix_tables": pages[:GROUPS * most_p].view(GROUPS, most_p).to(device),
        "tables": pages[GROUPS * most_p:GROUPS * most_p + n * most_s].view(n, most_s).to(device),
        "prefix_lens": torch.tensor(PREFIX, dtype=torch.int32, device=device),
        "group_starts": torch.tensor([0, EACH, 2 * EACH], dtype=torch.int32, device=device),
    }


def _prompts(m, table):
    import tome_b200
    device = m["prompt"].device
    place = torch.cat([torch.arange(x) for x in PREFIX]).to(torch.int32).to(device)
    owner = torch.repeat_interleave(torch.arange(GROUPS), torch.tensor(PREFIX)).to(torch.int32).to(device)
    tome_b200.qk_norm_rope_append(m["prompt"], m["qw"], m["kw"], table, place, m["k_pool"], m["v_pool"], m["prefix_tables"],
                                  place, seq_ids=owner, eps=EPS, check=True)


def _decode(m, table, x, place, rotary, lengths):
    import tome_b200
    q = tome_b200.qk_norm_rope_append(x, m["qw"], m["kw"], table, rotary, m["k_pool"], m["v_pool"], m["tables"], place, eps=EPS)
    out = tome_b200.shared_prefix_attention(q, m["k_pool"], m["v_pool"], m["prefix_tables"], m["prefix_lens"],
                                            m["group_starts"], m["tables"], lengths)
    return q, out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rollout_then_training(cuda_device, dtype):
    import tome_b200
    m = _model(cuda_device, dtype)
    table = tome_b200.rope_table(64, DIM, device=cuda_device)
    n = GROUPS * EACH
    before = torch.repeat_interleave(m["prefix_lens"], EACH).contiguous()
    _prompts(m, table)
    logits, outs = [], []
    for t in range(STEPS):
        place = torch.full((n,), t, dtype=torch.int32, device=cuda_device)
        q, out = _decode(m, table, m["tokens"][t], place, before + place, place + 1)
        outs.append(out)
        args = (q.cpu(), m["k_pool"].cpu(), m["v_pool"].cpu(), m["prefix_tables"].cpu(), m["prefix_lens"].cpu(),
                m["group_starts"].cpu(), m["tables"].cpu(), (place + 1).cpu())
        want, _, size, reach = step.attention(*args, DIM ** -0.5)
        u = torch.finfo(dtype).eps / 2
        tiny = 2.0 ** -24 * 32 * float(m["v_pool"].float().abs().max()) if dtype == torch.float16 else 0.0
        tol = u * want.abs() + (u + 2 * DIM * 2.0 ** -23 * reach[..., None] + 2.0 ** -14) * size + tiny + 1e-30
        assert bool(((out.cpu().double() - want).abs() <= tol).all())
        logits.append(out.reshape(n, HEADS * DIM) @ m["head"])
    # the cache holds what the training form computes for the same tokens, bit for bit
    whole = m["tokens"].transpose(0, 1).contiguous()                       # [n, STEPS, width]
    positions = (before[:, None] + torch.arange(STEPS, device=cuda_device, dtype=torch.int32)).contiguous()
    q, k = tome_b200.qk_norm_rope(whole, m["qw"], m["kw"], table, positions, HEADS, KV, eps=EPS, check=True)
    cached = m["k_pool"][m["tables"][:, 0].long()][:, :, :STEPS].transpose(1, 2)
    assert torch.equal(k, cached)
    values = whole.view(n, STEPS, HEADS + 2 * KV, DIM)[:, :, HEADS + KV:]
    assert torch.equal(values, m["v_pool"][m["tables"][:, 0].long()][:, :, :STEPS].transpose(1, 2))
    # sampled tokens, scored by the loss: the policy has not moved, so every ratio is 1
    x = torch.stack(logits, 1).to(torch.bfloat16)                           # [n, STEPS, VOCAB]
    tok, lp = tome_b200.sample_topk_logprob(x.reshape(n * STEPS, VOCAB).contiguous(), TEMP, 20, seed=1, offset=0)[:2]
    ids, old = tok.view(n, STEPS).to(torch.int32), lp.view(n, STEPS)
    adv = torch.tensor([1.0, -0.5, 0.25, -1.0, 0.0, 2.0], device=cuda_device)
    lengths = torch.tensor([5, 3, 0, 1, 5, 2], dtype=torch.int32, device=cuda_device)
    loss, scored, grad = tome_b200.grpo_policy_loss(x, ids, old, adv, lengths, TEMP, check=True)
    active = torch.arange(STEPS, device=cuda_device)[None] < lengths[:, None]
    assert bool(((scored - old).abs() <= 2.0 ** -16)[active].all()) and not bool(scored[~active].any())
    want = -(adv * lengths).sum() / lengths.sum()
    assert abs(float(loss) - float(want)) <= 2.0 ** -14 * float((adv.abs() * lengths).sum() / lengths.sum())
    assert not bool(grad[~active].any())
    # a row of the gradient sums to zero: V entries, each off by half a bf16 step and the p's rounding
    sums, sizes = grad.double().sum(-1), grad.double().abs().sum(-1)
    assert bool((sums.abs() <= (2.0 ** -8 + 2.0 ** -14) * sizes).all())
    # and the norm's gradient of the same tokens
    g = torch.Generator().manual_seed(6)
    dq, dk = (torch.randn(tuple(z.shape), generator=g).to(dtype).to(cuda_device) for z in (q, k))
    dx, dqw, dkw = tome_b200.qk_norm_rope_backward(dq, dk, whole, m["qw"], m["kw"], table, positions, eps=EPS, check=True)
    heads = whole.reshape(n * STEPS, HEADS + 2 * KV, DIM)
    got = dx.reshape(n * STEPS, HEADS + 2 * KV, DIM).cpu().double()
    for part, w, d, gw, at in ((heads[:, :HEADS], m["qw"], dq, dqw, slice(0, HEADS)),
                               (heads[:, HEADS:HEADS + KV], m["kw"], dk, dkw, slice(HEADS, HEADS + KV))):
        want, ww, size, wsize = step.norm_rope_backward(part, w, d.reshape(n * STEPS, -1, DIM), table, positions.reshape(-1), EPS)
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
        assert bool(((got[:, at] - want).abs() <= torch.finfo(dtype).eps / 2 * 1.001 * want.abs() + 64 * 2.0 ** -24 * size + tiny).all())
        assert bool(((gw.cpu().double() - ww).abs() <= 128 * 2.0 ** -24 * wsize + 1e-30).all())


def test_decoding_as_one_captured_step(cuda_device):
    """The step of a decode loop as a graph: places and lengths are counted on the device, the replays
    give what the calls gave one by one."""
    import tome_b200
    m = _model(cuda_device, torch.bfloat16)
    table = tome_b200.rope_table(64, DIM, device=cuda_device)
    n = GROUPS * EACH
    before = torch.repeat_interleave(m["prefix_lens"], EACH).contiguous()
    _prompts(m, table)
    empty = (m["k_pool"].clone(), m["v_pool"].clone())
    want = []
    for t in range(STEPS):
        place = torch.full((n,), t, dtype=torch.int32, device=cuda_device)
        want.append(_decode(m, table, m["tokens"][t], place, before + place, place + 1)[1])
    filled = (m["k_pool"].clone(), m["v_pool"].clone())
    x = m["tokens"][0].clone()
    place = torch.zeros(n, dtype=torch.int32, device=cuda_device)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _, out = _decode(m, table, x, place, before + place, place + 1)
        place += 1
    place.zero_()
    for dst, src in zip((m["k_pool"], m["v_pool"]), empty):
        dst.copy_(src)
    for t in range(STEPS):
        x.copy_(m["tokens"][t])
        graph.replay()
        assert torch.equal(out, want[t])
    assert torch.equal(m["k_pool"], filled[0]) and torch.equal(m["v_pool"], filled[1])
    tome_b200.check_device_status(cuda_device)
