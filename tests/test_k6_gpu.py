"""GPU tests of the query/key norm with rotation (forward, backward, append) against the 64-bit
oracle.  Tolerances: half a step of the output's type for the store, and for the fp32 arithmetic
2^-24 of what was added up times the length of the longest chain (the sum of squares: 16 products
per thread and at most four exchanges; the rest: under ten roundings), taken as 64."""
import pytest
import torch

from oracle import oracle, step

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    """Half a step of the smallest values (fp16 has few of them)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _inputs(tokens, heads, kv, dim, dtype, seed, positions=700):
    import tome_b200
    g = torch.Generator().manual_seed(seed)
    qkv = (1.5 * torch.randn((tokens, (heads + 2 * kv) * dim), generator=g)).to(dtype)
    qw = (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype)
    kw = (1 + 0.2 * torch.randn(dim, generator=g)).to(dtype)
    pos = torch.randint(0, positions, (tokens,), generator=g, dtype=torch.int32)
    return qkv, qw, kw, tome_b200.rope_table(positions, dim, device="cpu"), pos, g


def _close(got, want, size, dtype, chain=64):
    tol = _half_step(dtype) * want.abs() * 1.001 + chain * F32 * size + _tiny(dtype)
    bad = (got.cpu().double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got.cpu().double() - want).abs() / tol).max()))


SHAPES = [(1, 1, 1, 16), (3, 2, 1, 32), (5, 3, 1, 48), (8, 16, 8, 128), (33, 5, 5, 64), (7, 6, 2, 96),
          (130, 4, 2, 256), (1000, 16, 8, 128), (257, 24, 4, 80)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv,dim", SHAPES)
def test_forward(cuda_device, tokens, heads, kv, dim, dtype):
    import tome_b200
    qkv, qw, kw, table, pos, _ = _inputs(tokens, heads, kv, dim, dtype, tokens + dim)
    q, k = tome_b200.qk_norm_rope(*(x.to(cuda_device) for x in (qkv, qw, kw, table, pos)), heads, kv, check=True)
    x = qkv.view(tokens, heads + 2 * kv, dim)
    for got, part, w in ((q, x[:, :heads], qw), (k, x[:, heads:heads + kv], kw)):
        want, size = step.norm_rope(part, w, table, pos, 1e-6)
        assert got.shape == want.shape and got.dtype == dtype
        _close(got, want, size, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv,dim", SHAPES)
def test_backward(cuda_device, tokens, heads, kv, dim, dtype):
    import tome_b200
    qkv, qw, kw, table, pos, g = _inputs(tokens, heads, kv, dim, dtype, tokens + dim)
    dq, dk, dv = (torch.randn((tokens, n, dim), generator=g).to(dtype) for n in (heads, kv, kv))
    dev = [t.to(cuda_device) for t in (dq, dk, qkv, qw, kw, table, pos)]
    grad, gqw, gkw = tome_b200.qk_norm_rope_backward(*dev, grad_v=dv.to(cuda_device), check=True)
    again = tome_b200.qk_norm_rope_backward(*dev)
    x = qkv.view(tokens, heads + 2 * kv, dim)
    got = grad.view(tokens, heads + 2 * kv, dim)
    assert torch.equal(got[:, heads + kv:].cpu(), dv)
    assert not bool(again[0].view(tokens, -1, dim)[:, heads + kv:].any())       # no grad_v: zeros
    assert torch.equal(again[1], gqw) and torch.equal(again[2], gkw)            # the order is fixed
    for part, w, d, gx, gw in ((x[:, :heads], qw, dq, got[:, :heads], gqw),
                               (x[:, heads:heads + kv], kw, dk, got[:, heads:heads + kv], gkw)):
        dx, dw, size, wsize = step.norm_rope_backward(part, w, d, table, pos, 1e-6)
        _close(gx, dx, size, dtype)
        # a weight gradient: each term has under 64 roundings, their sum goes through at most
        # (heads a thread sees + 5 + 8 + 32 + 5) additions
        chain = 64 + 50 + tokens * heads // 64
        assert bool(((gw.cpu().double() - dw).abs() <= chain * F32 * wsize + 1e-30).all())


def test_strided_rows_leading_dims_and_out(cuda_device):
    import tome_b200
    heads, kv, dim = 4, 2, 64
    qkv, qw, kw, table, pos, _ = _inputs(30, heads, kv, dim, torch.bfloat16, 5)
    qkv, qw, kw, table, pos = (x.to(cuda_device) for x in (qkv, qw, kw, table, pos))
    q0, k0 = tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, heads, kv)
    wide = torch.full((30, qkv.shape[1] + 24), 7.0, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 8:8 + qkv.shape[1]] = qkv                     # a pitch, 16 bytes in: taken as it is
    odd = torch.full((30, qkv.shape[1] + 3), 7.0, dtype=torch.bfloat16, device=cuda_device)
    odd[:, 1:1 + qkv.shape[1]] = qkv                      # off the 16-byte grid: copied
    for view in (wide[:, 8:8 + qkv.shape[1]], odd[:, 1:1 + qkv.shape[1]], qkv.t().contiguous().t()):
        q, k = tome_b200.qk_norm_rope(view, qw, kw, table, pos.long(), heads, kv)
        assert torch.equal(q, q0) and torch.equal(k, k0)
    q, k = tome_b200.qk_norm_rope(qkv.view(5, 6, -1), qw, kw, table, pos.view(5, 6), heads, kv,
                                  out=(torch.empty((5, 6, heads, dim), dtype=torch.bfloat16, device=cuda_device),
                                       torch.empty((5, 6, kv, dim), dtype=torch.bfloat16, device=cuda_device)))
    assert torch.equal(q.view(30, heads, dim), q0) and torch.equal(k.view(30, kv, dim), k0)
    # no token
    q, k = tome_b200.qk_norm_rope(qkv[:0], qw, kw, table, pos[:0], heads, kv)
    assert q.shape == (0, heads, dim)
    g, a, b = tome_b200.qk_norm_rope_backward(q, k, qkv[:0], qw, kw, table, pos[:0])
    assert g.shape == qkv[:0].shape and not bool(a.any()) and not bool(b.any())


def test_bad_positions_and_refusals(cuda_device):
    import tome_b200
    heads, kv, dim = 2, 1, 64
    qkv, qw, kw, table, pos, _ = _inputs(6, heads, kv, dim, torch.bfloat16, 5, positions=40)
    qkv, qw, kw, table, pos = (x.to(cuda_device) for x in (qkv, qw, kw, table, pos))
    q0, _ = tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, heads, kv)
    bad = pos.clone()
    bad[1], bad[4] = 40, -1
    q, k = tome_b200.qk_norm_rope(qkv, qw, kw, table, bad, heads, kv)
    with pytest.raises(tome_b200.TomeRuntimeError, match="rotary"):
        tome_b200.check_device_status(cuda_device)
    assert bool(q[[1, 4]].isnan().all()) and bool(k[[1, 4]].isnan().all())
    assert torch.equal(q[[0, 2, 3, 5]], q0[[0, 2, 3, 5]])
    for call in (lambda: tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, 3, 1),
                 lambda: tome_b200.qk_norm_rope(qkv, qw[:32], kw, table, pos, heads, kv),
                 lambda: tome_b200.qk_norm_rope(qkv, qw, kw, table[:, :32], pos, heads, kv),
                 lambda: tome_b200.qk_norm_rope(qkv, qw, kw, table, pos[:-1], heads, kv),
                 lambda: tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, 0, 4),
                 lambda: tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, heads, kv, eps=-1.0),
                 lambda: tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, heads, kv,
                                                out=(qkv.view(6, 4, dim)[:, :2], q0)),
                 lambda: tome_b200.qk_norm_rope_backward(q0, q0[:, :1].contiguous(), qkv, qw, kw, table, pos,
                                                         out=qkv)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        tome_b200.qk_norm_rope(qkv.double(), qw, kw, table, pos, heads, kv)
    with pytest.raises(TypeError):
        tome_b200.qk_norm_rope(qkv, qw.float(), kw, table, pos, heads, kv)
    with pytest.raises(TypeError):
        tome_b200.qk_norm_rope(qkv, qw, kw, table, pos.float(), heads, kv)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block,seqs,each,heads,kv,dim", [(1, 3, 4, 2, 1, 64), (5, 4, 9, 6, 2, 48), (16, 8, 1, 16, 8, 128),
                                                          (16, 3, 70, 8, 4, 128), (24, 2, 33, 3, 3, 256)])
def test_append(cuda_device, block, seqs, each, heads, kv, dim, dtype):
    """Queries and cached keys equal the forward's, values are copied, nothing else is touched."""
    import tome_b200
    tokens = seqs * each
    qkv, qw, kw, table, pos, g = _inputs(tokens, heads, kv, dim, dtype, block + dim)
    first = torch.randint(0, 40, (seqs,), generator=g)
    at = (first[:, None] + torch.arange(each)).reshape(-1).to(torch.int32)
    sid = torch.arange(seqs).repeat_interleave(each).to(torch.int32)
    order = torch.randperm(tokens, generator=g)            # tokens in any order
    at, sid = at[order], sid[order]
    at[tokens // 2] = -1                                    # one token is not cached
    per = (40 + each + block - 1) // block
    tables = torch.randperm(seqs * per + 2, generator=g)[:seqs * per].view(seqs, per).to(torch.int32)
    pools = [torch.randn((seqs * per + 2, kv, block, dim), generator=g).to(dtype) for _ in range(2)]
    kp, vp = (x.to(cuda_device) for x in pools)
    dev = [x.to(cuda_device) for x in (qkv, qw, kw, table, pos)]
    one_each = each == 1
    if one_each:
        tables = tables[sid.long()]                        # token t is sequence t
    q = tome_b200.qk_norm_rope_append(*dev, kp, vp, tables.to(cuda_device), at.to(cuda_device),
                                      seq_ids=None if one_each else sid.to(cuda_device), check=True)
    q0, k0 = tome_b200.qk_norm_rope(*dev, heads, kv)
    assert torch.equal(q, q0)
    want_k, want_v = (x.clone() for x in pools)
    v = qkv.view(tokens, -1, dim)[:, heads + kv:]
    for t in range(tokens):
        if at[t] >= 0:
            row = t if one_each else int(sid[t])
            page, off = int(tables[row, int(at[t]) // block]), int(at[t]) % block
            want_k[page, :, off], want_v[page, :, off] = k0[t].cpu(), v[t]
    assert torch.equal(kp.cpu(), want_k) and torch.equal(vp.cpu(), want_v)


def test_append_skips_and_reports_bad_places(cuda_device):
    import tome_b200
    heads, kv, dim, block = 2, 1, 64, 4
    qkv, qw, kw, table, pos, g = _inputs(6, heads, kv, dim, torch.bfloat16, 9)
    dev = [x.to(cuda_device) for x in (qkv, qw, kw, table, pos)]
    pool = torch.randn((3, kv, block, dim), generator=g).to(torch.bfloat16).to(cuda_device)
    kp, vp = pool.clone(), pool.clone()
    tables = torch.tensor([[0, 3], [-1, 1], [2, 2]], dtype=torch.int32, device=cuda_device)
    sid = torch.tensor([0, 0, 1, 2, 3, -1], dtype=torch.int32, device=cuda_device)
    at = torch.tensor([4, 0, 0, 8, 0, 0], dtype=torch.int32, device=cuda_device)  # only token 1 has a place
    tome_b200.qk_norm_rope_append(*dev, kp, vp, tables, at, seq_ids=sid)
    with pytest.raises(tome_b200.TomeRuntimeError, match="block-table"):
        tome_b200.check_device_status(cuda_device)
    changed = (kp != pool).flatten(2).any(2).nonzero().tolist()
    assert changed == [[0, 0]]
    for i in range(1, 3):
        assert torch.equal(kp[i], pool[i]) and torch.equal(vp[i], pool[i])
    for call in (lambda: tome_b200.qk_norm_rope_append(*dev, kp, vp, tables, at),            # 6 tokens, 3 sequences
                 lambda: tome_b200.qk_norm_rope_append(*dev, kp, kp, tables, at, seq_ids=sid),
                 lambda: tome_b200.qk_norm_rope_append(*dev, kp, vp.half(), tables, at, seq_ids=sid),
                 lambda: tome_b200.qk_norm_rope_append(*dev, kp.transpose(1, 2), vp.transpose(1, 2), tables, at,
                                                       seq_ids=sid),
                 lambda: tome_b200.qk_norm_rope_append(*dev, kp, vp, tables[0], at, seq_ids=sid)):
        with pytest.raises(ValueError):
            call()


def test_append_then_gather_gives_the_keys_back(cuda_device):
    """The pool layout is that of gather_paged_kv."""
    import tome_b200
    heads, kv, dim, block, n = 4, 2, 64, 16, 37
    qkv, qw, kw, table, _, g = _inputs(n, heads, kv, dim, torch.bfloat16, 2)
    pos = torch.arange(n, dtype=torch.int32)
    dev = [x.to(cuda_device) for x in (qkv, qw, kw, table, pos)]
    kp = torch.zeros((8, kv, block, dim), dtype=torch.bfloat16, device=cuda_device)
    vp = torch.zeros_like(kp)
    tables = torch.tensor([[6, 1, 3]], dtype=torch.int32, device=cuda_device)
    zeros = torch.zeros(n, dtype=torch.int32, device=cuda_device)
    tome_b200.qk_norm_rope_append(*dev, kp, vp, tables, dev[4], seq_ids=zeros)
    _, k0 = tome_b200.qk_norm_rope(*dev, heads, kv)
    kg, vg = tome_b200.gather_paged_kv(tables, torch.tensor([n], device=cuda_device), kp, vp, n)
    assert torch.equal(kg[0].transpose(0, 1), k0)
    assert torch.equal(vg[0].transpose(0, 1).cpu(), qkv.view(n, -1, dim)[:, heads + kv:])


def test_rounding_of_the_norm_agrees_with_the_frameworks_rms_norm(cuda_device):
    """At position 0 the rotation is the identity: one head is what rms_norm gives."""
    import tome_b200
    g = torch.Generator().manual_seed(8)
    x = torch.randn((40, 3 * 128), generator=g).to(torch.bfloat16).to(cuda_device)
    w = (1 + 0.1 * torch.randn(128, generator=g)).to(torch.bfloat16).to(cuda_device)
    q, k = tome_b200.qk_norm_rope(x, w, w, tome_b200.rope_table(4, 128, device=cuda_device),
                                  torch.zeros(40, dtype=torch.int32, device=cuda_device), 1, 1)
    for got, part in ((q, x[:, :128]), (k, x[:, 128:256])):
        want = oracle.rms_norm(part.cpu(), w.cpu(), 1e-6)
        ours = tome_b200.rms_norm(part, w, 1e-6)
        # one bf16 step apart at most: each is within half a step of the same number
        assert bool(((got[:, 0].cpu().double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs()).all())
        assert bool(((got[:, 0].double() - ours.double()).abs() <= 2.0 ** -7 * ours.double().abs()).all())


def test_side_stream_and_captured_graph(cuda_device):
    import tome_b200
    heads, kv, dim = 8, 4, 128
    qkv, qw, kw, table, pos, g = _inputs(50, heads, kv, dim, torch.bfloat16, 5)
    qkv, qw, kw, table, pos = (x.to(cuda_device) for x in (qkv, qw, kw, table, pos))
    dq = torch.randn((50, heads, dim), generator=g).to(torch.bfloat16).to(cuda_device)
    dk = dq[:, :kv].contiguous()
    want = tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, heads, kv)
    want_g = tome_b200.qk_norm_rope_backward(dq, dk, qkv, qw, kw, table, pos)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        got = tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, heads, kv)
        got_g = tome_b200.qk_norm_rope_backward(dq, dk, qkv, qw, kw, table, pos)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want + want_g, got + got_g))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, heads, kv)
        got_g = tome_b200.qk_norm_rope_backward(dq, dk, qkv, qw, kw, table, pos)
    qkv.mul_(0.5).add_(0.25)
    graph.replay()
    torch.cuda.synchronize()
    want = tome_b200.qk_norm_rope(qkv, qw, kw, table, pos, heads, kv)
    want_g = tome_b200.qk_norm_rope_backward(dq, dk, qkv, qw, kw, table, pos)
    assert all(torch.equal(a, b) for a, b in zip(want + want_g, got + got_g))


@pytest.mark.parametrize("tokens,heads,kv,dim", [(1, 1, 1, 64), (400, 3, 1, 64), (401, 5, 3, 48), (333, 3, 3, 128)])
def test_backward_without_eps(cuda_device, tokens, heads, kv, dim):
    """Odd heads and tokens: what a group of threads does not have adds nothing to the weights' sums."""
    import tome_b200
    qkv, qw, kw, table, pos, g = _inputs(tokens, heads, kv, dim, torch.float32, tokens)
    dq, dk = (torch.randn((tokens, n, dim), generator=g) for n in (heads, kv))
    got = tome_b200.qk_norm_rope_backward(*(x.to(cuda_device) for x in (dq, dk, qkv, qw, kw, table, pos)), eps=0.0, check=True)
    x, dx = qkv.view(tokens, heads + 2 * kv, dim), got[0].view(tokens, heads + 2 * kv, dim)
    for part, w, d, at, gw in ((x[:, :heads], qw, dq, dx[:, :heads], got[1]),
                               (x[:, heads:heads + kv], kw, dk, dx[:, heads:heads + kv], got[2])):
        want, dw, size, wsize = step.norm_rope_backward(part, w, d, table, pos, 0.0)
        _close(at, want, size, torch.float32)
        chain = 64 + 50 + tokens * heads // 64
        assert bool(((gw.cpu().double() - dw).abs() <= chain * F32 * wsize + 1e-30).all())


def test_append_of_bad_positions_leaves_the_place_as_it_was(cuda_device):
    """Neither the key nor the value is cached: a place never holds a key of one token and a value of another."""
    import tome_b200
    heads, kv, dim, block, n = 2, 2, 64, 4, 5
    qkv, qw, kw, table, pos, g = _inputs(n, heads, kv, dim, torch.bfloat16, 9)
    pos[1], pos[3] = -1, table.shape[0]
    pool = torch.randn((n, kv, block, dim), generator=g).to(torch.bfloat16).to(cuda_device)
    kp, vp = pool.clone(), pool.clone()
    tables = torch.arange(n, dtype=torch.int32, device=cuda_device)[:, None].contiguous()
    at = torch.full((n,), 2, dtype=torch.int32, device=cuda_device)
    q = tome_b200.qk_norm_rope_append(*(x.to(cuda_device) for x in (qkv, qw, kw, table, pos)), kp, vp, tables, at)
    with pytest.raises(tome_b200.TomeRuntimeError, match="rotary"):
        tome_b200.check_device_status(cuda_device)
    assert q.isnan().flatten(1).all(1).tolist() == [False, True, False, True, False]
    for t in range(n):
        changed = t not in (1, 3)
        for p in (kp, vp):
            assert bool((p[t, :, 2] != pool[t, :, 2]).any()) == changed
            assert torch.equal(p[t, :, [0, 1, 3]], pool[t, :, [0, 1, 3]])
