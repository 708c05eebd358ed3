"""What is measured of the operators around the log-prob path: query/key norm with rotary
positions (forward, backward, append to the paged cache), attention over a paged cache whose
prefix is shared by a group, and the clipped policy loss with its gradient.

``run`` computes an operator either in elementary torch operations (``own = False``) or through
the framework's public entry points (``own = True``) on what ``prepare`` made.
"""
import math

import torch

own = False

EPS = 1e-6
ROPE_BASE = 1000000.0
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _norm(name, op, tokens, heads, kv_heads, head_dim, dtype):
    return {"name": name, "op": op, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype}


def _append(name, sequences, per_sequence, block, heads, kv_heads, head_dim, dtype):
    return {"name": name, "op": "append", "sequences": sequences, "per_sequence": per_sequence,
            "block": block, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype}


def _attention(name, groups, per_group, prefix, suffix, block, heads, kv_heads, head_dim, dtype):
    return {"name": name, "op": "attention", "groups": groups, "per_group": per_group,
            "prefix": prefix, "suffix": suffix, "block": block, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype}


def _loss(name, sequences, length, vocab, reduction, dtype):
    return {"name": name, "op": "loss", "sequences": sequences, "length": length, "vocab": vocab,
            "reduction": reduction, "dtype": dtype}


def listed():
    return [
        # one decode step of a small batch: 8 sequences, one token each (a launch's latency)
        _append("append_decode_8", 8, 1, 16, 16, 8, 128, "bf16"),
        # prompts of 4 requests written into the cache, an odd number of tokens each
        _append("append_prompts_4x1021", 4, 1021, 32, 32, 8, 128, "fp16"),
        # a training step's forward: 4 prompts x 8 completions x 640 tokens, 16 / 8 heads
        _norm("norm_rope_20480", "norm_rope", 20480, 16, 8, 128, "bf16"),
        # its backward pass
        _norm("norm_rope_backward_20480", "norm_rope_backward", 20480, 16, 8, 128, "bf16"),
        # a ragged micro-batch in full precision, small heads
        _norm("norm_rope_backward_1531_fp32", "norm_rope_backward", 1531, 12, 4, 64, "fp32"),
        # the first tokens of one prompt's completions: latency
        _attention("attention_1x8_short", 1, 8, 100, 24, 16, 16, 8, 128, "bf16"),
        # the rollout of 4 prompts x 8 completions of up to 640 tokens
        _attention("attention_4x8_rollout", 4, 8, 512, 640, 16, 16, 8, 128, "bf16"),
        # one long document, 64 short answers: the prefix is nearly all there is
        _attention("attention_1x64_document", 1, 64, 16381, 200, 32, 32, 8, 128, "fp16"),
        # long prompts and long completions
        _attention("attention_8x16_long", 8, 16, 8192, 2048, 64, 32, 8, 128, "bf16"),
        # the policy update of 32 completions of up to 256 tokens
        _loss("loss_32x256", 32, 256, 151936, "token", "bf16"),
        # a few tokens of one completion, 32-bit logits
        _loss("loss_1x24_fp32", 1, 24, 151936, "sequence", "fp32"),
        # a vocabulary off every grid
        _loss("loss_12x90_odd_vocabulary", 12, 90, 50257, "sequence", "bf16"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "norm_rope", "norm_rope_backward", "attention", "attention", "loss",
                     "loss"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (8, 8), (24, 4), (12, 4), (16, 1)])
    head_dim = rng.choice([64, 128, 128])
    while True:
        if op == "append":
            sequences, each = _spread(rng, 1, 256), _spread(rng, 1, 2048)
            case = _append("", sequences, each, rng.choice([8, 16, 24, 32, 64]), heads, kv_heads,
                           head_dim, rng.choice(["bf16", "fp16"]))
            fits = sequences * each <= 20480
        elif op == "attention":
            case = _attention("", rng.randint(1, 8), _spread(rng, 1, 64), _spread(rng, 1, 16384),
                              _spread(rng, 1, 2048), rng.choice([8, 16, 24, 32, 64]), heads,
                              kv_heads, head_dim, rng.choice(["bf16", "fp16"]))
            fits = (case["groups"] * (case["prefix"] + case["per_group"] * case["suffix"])
                    * kv_heads <= 8 * (8192 + 16 * 2048) * 8
                    and case["groups"] * case["per_group"] * heads
                    * (case["prefix"] + case["suffix"]) <= 128 * 32 * (8192 + 2048))
        elif op == "loss":
            vocab = rng.choice([151936, 128256, 50257, rng.randint(1000, 160000)])
            case = _loss("", rng.randint(1, 32), _spread(rng, 1, 512), vocab,
                         rng.choice(["token", "sequence"]), rng.choice(["bf16", "bf16", "fp32"]))
            fits = (case["sequences"] * case["length"] * vocab * BYTES[case["dtype"]]
                    <= 32 * 256 * 151936 * 2)
        else:
            case = _norm("", op, _spread(rng, 1, 20480), heads, kv_heads, head_dim,
                         rng.choice(["bf16", "bf16", "fp16", "fp32"]))
            fits = True
        if fits:
            break
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def _lengths(n, most):
    """n lengths from 1 to `most`, evenly spread: the same sum whatever their order."""
    return [most] if n == 1 else [1 + i * (most - 1) // (n - 1) for i in range(n)]


def _prefixes(case):
    """Prompt lengths of the groups: the named one and somewhat shorter ones."""
    return [max(1, case["prefix"] - g * (case["prefix"] // 16)) for g in range(case["groups"])]


def _rotary(positions, head_dim):
    """cos and sin of the angles, fp32 [positions, head_dim]: the table a model keeps."""
    half = head_dim // 2
    inv = ROPE_BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype="fp32"):
        return (scale * torch.randn(shape, generator=g, device="cuda")).to(TYPES[dtype])

    s = dict(case)
    dtype = case["dtype"]
    if case["op"] in ("norm_rope", "norm_rope_backward", "append"):
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        if case["op"] == "append":
            n, each, bs = case["sequences"], case["per_sequence"], case["block"]
            # where each sequence's cache ends: anywhere in a block
            first = torch.randint(0, 500, (n,), generator=g, device="cuda")
            at = (first[:, None] + torch.arange(each, device="cuda")).reshape(-1)
            s["tokens"] = n * each
            s["positions"] = at.to(torch.int32)
            s["sequence"] = torch.arange(n, device="cuda").repeat_interleave(each).to(torch.int32)
            per = (500 + each + bs - 1) // bs
            s["tables"] = torch.randperm(n * per, generator=g, device="cuda").view(n, per).to(
                torch.int32)
            s["k_pool"] = normal(n * per, kv, bs, d, dtype=dtype)
            s["v_pool"] = normal(n * per, kv, bs, d, dtype=dtype)
            s["table"] = _rotary(500 + each, d)
        else:
            s["positions"] = torch.randint(0, 4096, (case["tokens"],), generator=g,
                                           device="cuda").to(torch.int32)
            s["table"] = _rotary(4096, d)
        t = s["tokens"]
        # a projection's output; norm weights around one
        s["qkv"] = normal(t, (h + 2 * kv) * d, scale=1.5, dtype=dtype)
        s["q_weight"] = (1.0 + normal(d, scale=0.2)).to(TYPES[dtype])
        s["k_weight"] = (1.0 + normal(d, scale=0.2)).to(TYPES[dtype])
        if case["op"] == "norm_rope_backward":
            s["grad_q"] = normal(t, h, d, scale=0.01, dtype=dtype)
            s["grad_k"] = normal(t, kv, d, scale=0.01, dtype=dtype)
            s["grad_v"] = normal(t, kv, d, scale=0.01, dtype=dtype)
    elif case["op"] == "attention":
        h, kv, d, bs = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
        n = case["groups"] * case["per_group"]
        prefix = _prefixes(case)
        order = torch.randperm(n, generator=g, device="cuda")
        s["prefix_lens"] = _ints(prefix)
        s["suffix_lens"] = _ints(_lengths(n, case["suffix"]))[order].contiguous()
        s["group_starts"] = _ints([i * case["per_group"] for i in range(case["groups"] + 1)])
        most_p = (case["prefix"] + bs - 1) // bs
        most_s = (case["suffix"] + bs - 1) // bs
        blocks = case["groups"] * most_p + n * most_s
        pages = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        s["prefix_tables"] = pages[:case["groups"] * most_p].view(case["groups"], most_p)
        s["tables"] = pages[case["groups"] * most_p:].view(n, most_s)
        # normed and rotated queries and keys; some rows attend sharply
        s["q"] = normal(n, h, d, scale=2.0, dtype=dtype)
        s["k_pool"] = normal(blocks, kv, bs, d, dtype=dtype)
        s["v_pool"] = normal(blocks, kv, bs, d, dtype=dtype)
    else:
        n, length, vocab = case["sequences"], case["length"], case["vocab"]
        rows = n * length
        order = torch.randperm(n, generator=g, device="cuda")
        s["lengths"] = _ints(_lengths(n, length))[order].contiguous()
        # rollout logits with one column per row that stands out; 7 of 10 tokens drawn are it
        logits = torch.randn((rows, vocab), generator=g, device="cuda").mul_(3.0)
        best = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        logits[torch.arange(rows, device="cuda"), best] = 12.0
        other = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        ids = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.7, best, other)
        s["logits"] = logits.to(TYPES[dtype]).view(n, length, vocab)
        s["ids"] = ids.to(torch.int32).view(n, length)
        # the rollout's and the reference model's log-probs, near the policy's (and not within
        # rounding of the clip, where either side's gradient is right)
        del logits
        now = _log_probs(s["logits"].view(rows, vocab), ids, 0.9).view(n, length)
        drift = normal(n, length, scale=0.12)
        edge = ((drift - math.log(1.25)).abs() < 1e-3) | ((drift - math.log(0.8)).abs() < 1e-3)
        s["old"] = now - torch.where(edge, drift + 0.01, drift)
        s["ref"] = now + normal(n, length, scale=0.2)
        s["advantages"] = normal(n)
        s["temp"], s["clip"], s["kl_coef"] = 0.9, (0.2, 0.25), 0.04
    return s


def _log_probs(x, ids, temp):
    """Log-probs of ids: inputs that a rollout would have left, in 32 bits."""
    z = x.float() / temp
    top = z.amax(1)
    z = z.sub_(top[:, None]).exp_().sum(1)
    return x.gather(1, ids[:, None])[:, 0].float() / temp - top - z.log()


# ------------------------------------------------------------------ plain forms
def _plain_rotate(y, table, positions, back=False):
    half = y.shape[-1] // 2
    rows = table[positions.long()]
    cos, sin = rows[:, None, :half], rows[:, None, half:]
    sin = -sin if back else sin
    a, b = y[..., :half], y[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_split(s):
    t, h, kv, d = s["tokens"], s["heads"], s["kv_heads"], s["head_dim"]
    x = s["qkv"].float().view(t, h + 2 * kv, d)
    return x[:, :h], x[:, h:h + kv], x[:, h + kv:]


def _plain_norm_rope(s):
    q, k, _ = _plain_split(s)
    dtype = s["qkv"].dtype
    q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * s["q_weight"].float()
    k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * s["k_weight"].float()
    return (_plain_rotate(q, s["table"], s["positions"]).to(dtype),
            _plain_rotate(k, s["table"], s["positions"]).to(dtype))


def _plain_back(x, weight, grad, s):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    dy = _plain_rotate(grad.float(), s["table"], s["positions"], back=True)
    n = x * r
    gw = dy * weight.float()
    dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
    return dx, (dy * n).sum((0, 1))


def _plain_norm_rope_backward(s):
    q, k, _ = _plain_split(s)
    dq, dqw = _plain_back(q, s["q_weight"], s["grad_q"], s)
    dk, dkw = _plain_back(k, s["k_weight"], s["grad_k"], s)
    dqkv = torch.cat([dq, dk, s["grad_v"].float()], dim=1)
    return dqkv.view(s["tokens"], -1).to(s["qkv"].dtype), dqw, dkw


def _plain_append(s):
    q, k = _plain_norm_rope(s)
    v = s["qkv"].view(s["tokens"], -1, s["head_dim"])[:, s["heads"] + s["kv_heads"]:]
    at, bs = s["positions"].long(), s["block"]
    page = s["tables"].long()[s["sequence"].long(), at // bs]
    s["k_pool"][page, :, at % bs] = k
    s["v_pool"][page, :, at % bs] = v
    return q, s["k_pool"], s["v_pool"]


def _plain_pages(pool, tables):
    """[rows, kv_heads, tokens, head_dim] of the pages that each row of `tables` names."""
    x = pool[tables.long()].float()
    n, b, kv, bs, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(n, kv, b * bs, d)


def _plain_attention(s):
    n, h, d = s["q"].shape
    kv, gr, per = s["kv_heads"], s["groups"], s["per_group"]
    r = h // kv
    q = s["q"].float() * d ** -0.5
    k1, v1 = _plain_pages(s["k_pool"], s["prefix_tables"]), _plain_pages(s["v_pool"], s["prefix_tables"])
    k2, v2 = _plain_pages(s["k_pool"], s["tables"]), _plain_pages(s["v_pool"], s["tables"])
    q1 = q.view(gr, per, kv, r, d).transpose(1, 2).reshape(gr, kv, per * r, d)
    s1 = q1 @ k1.transpose(2, 3)
    s2 = q.view(n, kv, r, d) @ k2.transpose(2, 3)
    beyond1 = torch.arange(k1.shape[2], device="cuda") >= s["prefix_lens"][:, None]
    beyond2 = torch.arange(k2.shape[2], device="cuda") >= s["suffix_lens"][:, None]
    s1 = s1.masked_fill(beyond1[:, None, None], -math.inf)
    s2 = s2.masked_fill(beyond2[:, None, None], -math.inf)
    top2 = s2.amax(-1)
    top1 = s1.amax(-1).reshape(gr, kv, per, r).transpose(1, 2).reshape(n, kv, r)
    top = torch.maximum(top1, top2)
    e1 = (s1 - top.reshape(gr, per, kv, r).transpose(1, 2).reshape(gr, kv, per * r, 1)).exp()
    e2 = (s2 - top[..., None]).exp()
    o1 = (e1 @ v1).reshape(gr, kv, per, r, d).transpose(1, 2).reshape(n, kv, r, d)
    l1 = e1.sum(-1).reshape(gr, kv, per, r).transpose(1, 2).reshape(n, kv, r)
    total = l1 + e2.sum(-1)
    o = (o1 + e2 @ v2) / total[..., None]
    return o.reshape(n, h, d).to(s["q"].dtype), (top + total.log()).reshape(n, h)


def _plain_loss(s):
    n, length, vocab = s["logits"].shape
    temp, (low, high), kl_coef = s["temp"], s["clip"], s["kl_coef"]
    z = s["logits"].float() / temp
    top = z.amax(-1, keepdim=True)
    z = z - top
    ids = s["ids"].long()[..., None]
    drawn = z.gather(-1, ids)[..., 0]
    p = z.exp_()
    total = p.sum(-1)
    lp = drawn - total.log()
    adv = s["advantages"][:, None]
    ratio = (lp - s["old"]).exp()
    clipped = ratio.clamp(1 - low, 1 + high)
    away = s["ref"] - lp
    each = -torch.minimum(ratio * adv, clipped * adv) + kl_coef * (torch.expm1(away) - away)
    active = torch.arange(length, device="cuda") < s["lengths"][:, None]
    if s["reduction"] == "token":
        weight = active.float() / s["lengths"].sum()
    else:
        weight = active.float() / (n * s["lengths"][:, None])
    loss = (each.double() * weight).sum().float()
    slope = -adv * ratio * (ratio * adv <= clipped * adv) - kl_coef * torch.expm1(away)
    slope = slope * weight / temp
    p.mul_((-slope / total)[..., None])
    p.scatter_add_(-1, ids, slope[..., None])
    return loss, lp * active, p.to(s["logits"].dtype)


# ------------------------------------------------------------------ the framework's calls
def _kernels(s):
    import tome_b200 as tb
    if s["op"] == "append":
        q = tb.qk_norm_rope_append(
            s["qkv"], s["q_weight"], s["k_weight"], s["table"], s["positions"], s["k_pool"],
            s["v_pool"], s["tables"], s["positions"], seq_ids=s["sequence"], eps=EPS)
        return q, s["k_pool"], s["v_pool"]
    if s["op"] == "norm_rope":
        return tb.qk_norm_rope(s["qkv"], s["q_weight"], s["k_weight"], s["table"], s["positions"],
                               s["heads"], s["kv_heads"], eps=EPS)
    if s["op"] == "norm_rope_backward":
        return tb.qk_norm_rope_backward(
            s["grad_q"], s["grad_k"], s["qkv"], s["q_weight"], s["k_weight"], s["table"],
            s["positions"], grad_v=s["grad_v"], eps=EPS)
    if s["op"] == "attention":
        return tb.shared_prefix_attention(
            s["q"], s["k_pool"], s["v_pool"], s["prefix_tables"], s["prefix_lens"],
            s["group_starts"], s["tables"], s["suffix_lens"], return_lse=True)
    return tb.grpo_policy_loss(
        s["logits"], s["ids"], s["old"], s["advantages"], s["lengths"], s["temp"],
        ref_logprobs=s["ref"], clip_low=s["clip"][0], clip_high=s["clip"][1],
        kl_coef=s["kl_coef"], reduction=s["reduction"])


def run(state):
    if own:
        return _kernels(state)
    return {"append": _plain_append, "norm_rope": _plain_norm_rope,
            "norm_rope_backward": _plain_norm_rope_backward, "attention": _plain_attention,
            "loss": _plain_loss}[state["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] in ("norm_rope", "norm_rope_backward", "append"):
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        if case["op"] == "append":
            t = case["sequences"] * case["per_sequence"]
            moved, flops = 2 * (h + 2 * kv) * d * b + 12, 9 * (h + kv) * d
            rotary = 4 * d * min(t, 500 + case["per_sequence"])
        else:
            t = case["tokens"]
            rotary = 4 * d * min(t, 4096)
            if case["op"] == "norm_rope":
                moved, flops = 2 * (h + kv) * d * b + 4, 9 * (h + kv) * d
            else:
                moved = (2 * (h + kv) + 2 * kv + (h + kv)) * d * b + 4
                flops = 20 * (h + kv) * d
        return {"bytes": t * moved + rotary + 4 * d * b, "flops": t * flops}
    if case["op"] == "attention":
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        n = case["groups"] * case["per_group"]
        suffix = sum(_lengths(n, case["suffix"]))
        prefix = _prefixes(case)
        pairs = h * (suffix + case["per_group"] * sum(prefix))
        return {"bytes": (suffix + sum(prefix)) * kv * d * 2 * b + n * h * (2 * d * b + 4),
                "flops": 4 * d * pairs}
    rows, active = case["sequences"] * case["length"], sum(_lengths(case["sequences"], case["length"]))
    return {"bytes": (rows + active) * case["vocab"] * b + 16 * rows,
            "flops": 8 * active * case["vocab"]}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_turn(head, table, positions, sign):
    half = head.shape[-1] // 2
    z = torch.complex(head[..., :half], head[..., half:])
    w = torch.complex(table[:, :half].double(), sign * table[:, half:].double())[positions.long()]
    z = z * w[:, None]
    return torch.cat([z.real, z.imag], dim=-1)


def _exact_norm(x, weight):
    return x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm_rope", "norm_rope_backward", "append"):
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        t = s["tokens"]
        q, k, v = s["qkv"].double().view(t, -1, d).split([h, kv, kv], dim=1)
        if case["op"] == "norm_rope_backward":
            found = []
            for x, weight, grad in ((q, "q_weight", "grad_q"), (k, "k_weight", "grad_k")):
                x = x.clone().requires_grad_()
                w = s[weight].double().requires_grad_()
                y = _exact_turn(_exact_norm(x, w), s["table"], s["positions"], 1.0)
                found.append(torch.autograd.grad(y, (x, w), s[grad].double()))
            (dq, dqw), (dk, dkw) = found
            return torch.cat([dq, dk, s["grad_v"].double()], dim=1).view(t, -1), dqw, dkw
        q = _exact_turn(_exact_norm(q, s["q_weight"]), s["table"], s["positions"], 1.0)
        k = _exact_turn(_exact_norm(k, s["k_weight"]), s["table"], s["positions"], 1.0)
        if case["op"] == "norm_rope":
            return q, k
        bs, at = case["block"], s["positions"].long()
        pools = []
        slot = s["tables"].long()[s["sequence"].long(), at // bs] * bs + at % bs
        for pool, new in ((s["k_pool"], k), (s["v_pool"], v)):
            flat = pool.double().transpose(1, 2).reshape(-1, kv, d)
            flat[slot] = new
            pools.append(flat.view(-1, bs, kv, d).transpose(1, 2).contiguous())
        return q, pools[0], pools[1]
    if case["op"] == "attention":
        n, h, d = s["q"].shape
        kv, bs = case["kv_heads"], case["block"]
        out = torch.empty((n, h, d), dtype=torch.float64, device="cuda")
        lse = torch.empty((n, h), dtype=torch.float64, device="cuda")
        for b in range(n):
            g = b // case["per_group"]
            kept = []
            for pool in (s["k_pool"], s["v_pool"]):
                rows = []
                for table, length in ((s["prefix_tables"][g], int(s["prefix_lens"][g])),
                                      (s["tables"][b], int(s["suffix_lens"][b]))):
                    pages = table[:(length + bs - 1) // bs].long()
                    rows.append(pool[pages].double().transpose(1, 2).reshape(-1, kv, d)[:length])
                kept.append(torch.cat(rows))
            score = torch.einsum("krd,tkd->krt", s["q"][b].double().view(kv, h // kv, d), kept[0])
            score = score / math.sqrt(d)
            lse[b] = torch.logsumexp(score, -1).reshape(h)
            out[b] = torch.einsum("krt,tkd->krd", torch.softmax(score, -1), kept[1]).reshape(h, d)
        return out, lse
    n, length, vocab = s["logits"].shape
    grad = torch.zeros((n, length, vocab), dtype=torch.float64, device="cuda")
    lps = torch.zeros((n, length), dtype=torch.float64, device="cuda")
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    tokens = int(s["lengths"].sum())
    for i in range(n):
        m = int(s["lengths"][i])
        x = torch.log_softmax(s["logits"][i, :m].double() / s["temp"], -1)
        ids = s["ids"][i, :m].long()
        lp = x.gather(1, ids[:, None])[:, 0].requires_grad_()
        ratio = torch.exp(lp - s["old"][i, :m].double())
        a = s["advantages"][i].double()
        kept = torch.clamp(ratio, 1 - s["clip"][0], 1 + s["clip"][1])
        d = s["ref"][i, :m].double() - lp
        per = torch.maximum(-ratio * a, -kept * a) + s["kl_coef"] * (d.exp() - d - 1)
        part = per.sum() / (tokens if case["reduction"] == "token" else n * m)
        (slope,) = torch.autograd.grad(part, lp)
        loss += part.detach()
        lps[i, :m] = lp.detach()
        grad[i, :m] = -(slope / s["temp"])[:, None] * x.exp()
        grad[i, :m].scatter_add_(1, ids[:, None], (slope / s["temp"])[:, None])
    return loss, lps, grad
