"""GPU tests of the shared-prefix paged attention against the 64-bit oracle.

Tolerances, for a row with probabilities p, A = sum p |v| and u half a step of the type: u |out|
for the store; u A for the probabilities, each rounded to the type (an fp16 one below its normal
range: 2^-25 absolute, against a sum of at least 1/2); a score is a sum of D products in fp32, off
by at most D 2^-23 of |q||k| scale =: e (whatever the order, with one more bit for an accumulator
that truncates), which moves numerator and sum by e each; ex2 and the sums of up to 64 keys, then of
the tiles, then of the pieces: 2^-14."""
import pytest
import torch

from oracle import step

pytestmark = pytest.mark.gpu


def _case(seed, groups, lengths, prefix, block, heads, kv, dim, dtype, q_scale=2.0, spare=3):
    """`groups`: sizes; the sequences lie group after group."""
    g = torch.Generator().manual_seed(seed)
    n = len(lengths)
    most_p = max([1] + [(x + block - 1) // block for x in prefix])
    most_s = max([1] + [(x + block - 1) // block for x in lengths])
    used = len(groups) * most_p + n * most_s
    pages = torch.randperm(used + spare, generator=g)[:used].to(torch.int32)
    starts = [0]
    for x in groups:
        starts.append(starts[-1] + x)
    c = {
        "q": (q_scale * torch.randn((n, heads, dim), generator=g)).to(dtype),
        "k_pool": torch.randn((used + spare, kv, block, dim), generator=g).to(dtype),
        "v_pool": torch.randn((used + spare, kv, block, dim), generator=g).to(dtype),
        "prefix_tables": pages[:len(groups) * most_p].view(len(groups), most_p) if groups else None,
        "prefix_lens": torch.tensor(prefix, dtype=torch.int32) if groups else None,
        "group_starts": torch.tensor(starts, dtype=torch.int32) if groups else None,
        "tables": pages[len(groups) * most_p:].view(n, most_s),
        "lengths": torch.tensor(lengths, dtype=torch.int32),
    }
    return c


ORDER = ("q", "k_pool", "v_pool", "prefix_tables", "prefix_lens", "group_starts", "tables", "lengths")


def _dev(c, device):
    return [None if c[k] is None else c[k].to(device) for k in ORDER]


def _compare(c, out, lse, scale=None):
    dim, dtype = c["q"].shape[2], c["q"].dtype
    scale = dim ** -0.5 if scale is None else scale
    want, want_lse, size, reach = step.attention(*(c[k] for k in ORDER), scale)
    u = torch.finfo(dtype).eps / 2
    e = dim * 2.0 ** -23 * reach
    vmax = float(c["v_pool"].float().nan_to_num().abs().max())
    keys = int(c["lengths"].max()) + (int(c["prefix_lens"].max()) if c["prefix_lens"] is not None else 0)
    tiny = keys * 2.0 ** -24 * vmax if dtype == torch.float16 else 0.0
    tol = u * want.abs() + (u + 2 * e[..., None] + 2.0 ** -14) * size + tiny + 1e-30
    off = (out.cpu().double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    assert torch.equal(torch.isinf(lse.cpu()), torch.isinf(want_lse))
    fine = ~torch.isinf(want_lse)
    tol = e + 2.0 ** -14 + 2.0 ** -20 * want_lse.abs()
    assert bool(((lse.cpu().double() - want_lse).abs() <= tol)[fine].all())


def _run(c, device, **kw):
    import tome_b200
    out, lse = tome_b200.shared_prefix_attention(*_dev(c, device), return_lse=True, check=True, **kw)
    _compare(c, out, lse, kw.get("scale"))
    return out, lse


def test_one_tile(cuda_device):
    """One sequence, one head, keys within one tile."""
    _run(_case(1, [], [64], [], 16, 1, 1, 128, torch.bfloat16), cuda_device)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 127, 129, 200, 640])
def test_lengths(cuda_device, length, dtype, dim):
    _run(_case(length, [], [length, max(1, length - 1)], [], 16, 2, 1, dim, dtype), cuda_device)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (8, 2), (12, 2), (24, 4), (16, 1), (40, 1), (128, 1), (5, 5)])
def test_head_layouts(cuda_device, heads, kv, dim):
    _run(_case(heads, [3, 2], [5, 70, 130, 1, 64], [100, 65], 16, heads, kv, dim, torch.bfloat16), cuda_device)


@pytest.mark.parametrize("block", [1, 3, 8, 16, 24, 64, 100, 256])
def test_page_sizes(cuda_device, block):
    """Pages that end inside a tile, tiles that end inside a page."""
    _run(_case(block, [2, 1], [5, 150, 77], [131, 64], block, 4, 2, 64, torch.float16), cuda_device)


@pytest.mark.parametrize("sizes,rows", [([40], 4), ([33, 1, 70], 4), ([129], 1), ([64, 64], 2), ([3], 96)])
def test_groups_beyond_one_row_block(cuda_device, sizes, rows):
    """More query rows per KV head than the 128 of an item."""
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 90, (sum(sizes),), generator=g).tolist()
    _run(_case(3, sizes, lens, [200 - 30 * i for i in range(len(sizes))], 16, 2 * rows, 2, 64, torch.bfloat16), cuda_device)


def test_empty_prefixes_suffixes_groups_and_rows(cuda_device):
    """Rows that see nothing give 0 and -inf; groups and sequences may be empty."""
    c = _case(5, [2, 0, 2, 1], [0, 3, 0, 0, 70], [0, 50, 65, 0], 16, 4, 2, 128, torch.bfloat16)
    out, lse = _run(c, cuda_device)
    assert not bool(out[0].any()) and bool(torch.isinf(lse[0]).all())
    # sequences outside every group have no prefix
    c = _case(6, [2], [10, 20, 30, 0, 40], [33], 16, 4, 2, 128, torch.bfloat16)
    c["group_starts"] = torch.tensor([1, 3], dtype=torch.int32)
    _run(c, cuda_device)
    # no key anywhere
    c = _case(7, [2], [0, 0], [0], 16, 4, 2, 64, torch.bfloat16)
    out, lse = _run(c, cuda_device)
    assert not bool(out.any())


def test_long_prefix_is_split_over_many_ctas(cuda_device):
    for kv, heads in ((1, 2), (2, 8)):
        _run(_case(11, [4], [1, 30, 64, 200], [20011], 64, heads, kv, 128, torch.bfloat16), cuda_device)
    _run(_case(12, [], [9001], [], 16, 1, 1, 64, torch.float16), cuda_device)


def test_many_short_sequences(cuda_device):
    """More items than CTAs: a CTA's run of tiles holds many pieces."""
    g = torch.Generator().manual_seed(4)
    lens = torch.randint(0, 40, (700,), generator=g).tolist()
    _run(_case(13, [350, 350], lens, [70, 3], 8, 4, 2, 64, torch.bfloat16), cuda_device)


def test_scores_far_apart_and_scale(cuda_device):
    c = _case(14, [2], [100, 90], [150], 16, 4, 2, 128, torch.bfloat16, q_scale=20.0)
    _run(c, cuda_device)
    _run(c, cuda_device, scale=0.5)
    c["q"].zero_()                                        # every key alike
    _run(c, cuda_device)


def test_what_lies_behind_the_last_key_is_not_read(cuda_device):
    """NaN and infinities in masked places: in the rest of a page, in pages that no table names and in
    the tables' unused entries."""
    import tome_b200
    c = _case(15, [2], [5, 70], [37], 16, 4, 2, 64, torch.bfloat16)
    want = _run(c, cuda_device)
    k, v = c["k_pool"].clone(), c["v_pool"].clone()
    live = torch.zeros(k.shape[0], 16, dtype=torch.bool)
    for table, length in [(c["prefix_tables"][0], 37), (c["tables"][0], 5), (c["tables"][1], 70)]:
        for i in range(length):
            live[int(table[i // 16]), i % 16] = True
    k.permute(0, 2, 1, 3)[~live] = float("nan")
    v.permute(0, 2, 1, 3)[~live] = float("inf")
    tables, prefix = c["tables"].clone(), c["prefix_tables"].clone()
    tables[0, 1:] = -7
    d = _dev(dict(c, k_pool=k, v_pool=v, tables=tables, prefix_tables=prefix), cuda_device)
    out, lse = tome_b200.shared_prefix_attention(*d, return_lse=True, check=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_nan_stays_in_its_row(cuda_device):
    import tome_b200
    c = _case(16, [3], [5, 70, 20], [37], 16, 4, 2, 64, torch.bfloat16)
    want = _run(c, cuda_device)[0]
    c["q"][1, 2] = float("nan")
    out = tome_b200.shared_prefix_attention(*_dev(c, cuda_device))
    assert bool(out[1, 2].isnan().all())
    keep = torch.ones((3, 4), dtype=torch.bool)
    keep[1, 2] = False
    assert torch.equal(out.cpu()[keep], want.cpu()[keep])


def test_bad_pages_read_as_zeros_and_are_reported(cuda_device):
    import tome_b200
    c = _case(17, [2], [40, 20], [50], 16, 4, 2, 64, torch.bfloat16)
    c["tables"][0, 1] = 10 ** 6
    c["prefix_tables"][0, 2] = -1
    out, lse = tome_b200.shared_prefix_attention(*_dev(c, cuda_device), return_lse=True)
    with pytest.raises(tome_b200.TomeRuntimeError, match="block-table"):
        tome_b200.check_device_status(cuda_device)
    _compare(c, out, lse)
    # lengths past the tables: the tables' own; negative ones: none
    c = _case(18, [2], [40, 20], [50], 16, 4, 2, 64, torch.bfloat16)
    c["lengths"] = torch.tensor([1000, -5], dtype=torch.int32)
    c["prefix_lens"] = torch.tensor([2 ** 31 - 1], dtype=torch.int32)
    out, lse = tome_b200.shared_prefix_attention(*_dev(c, cuda_device), return_lse=True)
    with pytest.raises(tome_b200.TomeRuntimeError, match="block-table"):
        tome_b200.check_device_status(cuda_device)
    _compare(c, out, lse)
    # group_starts that are out of range or fall: clamped, every sequence in the group before it
    c = _case(19, [1, 1], [10, 20, 30], [50, 40], 16, 4, 2, 64, torch.bfloat16)
    d = _dev(c, cuda_device)
    d[5] = torch.tensor([-3, 2, 99], dtype=torch.int32, device=cuda_device)
    out, lse = tome_b200.shared_prefix_attention(*d, return_lse=True, check=True)
    c["group_starts"] = torch.tensor([0, 2, 3], dtype=torch.int32)
    _compare(c, out, lse)


def test_outputs_strides_workspace_and_repetition(cuda_device):
    import tome_b200
    c = _case(20, [4, 4], [5, 70, 20, 33, 1, 0, 128, 64], [300, 77], 16, 8, 2, 128, torch.bfloat16)
    want, want_lse = _run(c, cuda_device)
    d = _dev(c, cuda_device)
    n, heads, dim = c["q"].shape
    wide = torch.zeros((n, (heads + 4) * dim), dtype=torch.bfloat16, device=cuda_device)
    wide[:, :heads * dim] = d[0].reshape(n, -1)
    odd = torch.zeros((n, heads * dim + 1), dtype=torch.bfloat16, device=cuda_device)
    odd[:, 1:] = d[0].reshape(n, -1)
    out, lse = torch.empty_like(want), torch.empty_like(want_lse)
    ws = torch.full((tome_b200.shared_prefix_attention_workspace_bytes(n, 2, heads, 2, dim),), 255, dtype=torch.uint8,
                    device=cuda_device)                    # no initialisation is counted on
    for q in (d[0], wide[:, :heads * dim].view(n, heads, dim), odd[:, 1:].view(n, heads, dim),
              d[0].transpose(1, 2).contiguous().transpose(1, 2)):
        out.fill_(7), lse.fill_(7)
        got = tome_b200.shared_prefix_attention(q, *d[1:], out=out, out_lse=lse, workspace=ws)
        assert got[0].data_ptr() == out.data_ptr() and got[1].data_ptr() == lse.data_ptr()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert torch.equal(tome_b200.shared_prefix_attention(*d[:6], d[6].long(), d[7].long()), want)
    empty = tome_b200.shared_prefix_attention(d[0][:0], d[1], d[2], None, None, None, d[6][:0], d[7][:0])
    assert empty.shape == (0, heads, dim)


def test_streams_and_graphs(cuda_device):
    """Two calls at once on two streams, and a captured one replayed with other lengths (the split is
    made on the device)."""
    import tome_b200
    cases = [_case(21 + i, [3, 2], [5, 70, 200, 33, 1], [300, 77], 16, 8, 2, 128, torch.bfloat16) for i in range(2)]
    devs = [_dev(c, cuda_device) for c in cases]
    want = [tome_b200.shared_prefix_attention(*d) for d in devs]
    streams = [torch.cuda.Stream(cuda_device) for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tome_b200.shared_prefix_attention(*devs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
    d = devs[0]
    d[6] = d[6].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tome_b200.shared_prefix_attention(*d)
    for lens, prefix in (([1, 2, 208, 0, 150], [1, 304]), ([0, 0, 0, 0, 0], [5, 0]), ([200, 200, 7, 208, 65], [303, 64])):
        d[7].copy_(torch.tensor(lens, dtype=torch.int32))
        d[4].copy_(torch.tensor(prefix, dtype=torch.int32))
        out.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        eager, lse = tome_b200.shared_prefix_attention(*d, return_lse=True, check=True)
        assert torch.equal(out, eager)
        _compare(dict(cases[0], lengths=d[7].cpu(), prefix_lens=d[4].cpu()), eager, lse)


def test_refusals(cuda_device):
    import tome_b200
    c = _case(30, [2], [40, 20], [50], 16, 4, 2, 64, torch.bfloat16)
    d = _dev(c, cuda_device)

    def call(**kw):
        a = list(d)
        for k, v in kw.items():
            if k in ORDER:
                a[ORDER.index(k)] = v
        return tome_b200.shared_prefix_attention(*a, **{k: v for k, v in kw.items() if k not in ORDER})
    for kw in ({"q": d[0][0]}, {"k_pool": d[1][:, :1].contiguous()}, {"k_pool": d[1].half(), "v_pool": d[2].half()},
               {"k_pool": d[1].transpose(1, 2), "v_pool": d[2].transpose(1, 2)}, {"tables": d[6][:1]},
               {"lengths": d[7][:1]}, {"prefix_lens": None}, {"group_starts": d[5][:1]}, {"prefix_tables": d[3][0]},
               {"prefix_tables": None}, {"scale": 0.0}, {"scale": float("nan")}, {"out": d[0]}, {"out": d[0][:1]},
               {"out_lse": torch.zeros((2, 3), device=cuda_device)}, {"q": d[0][:, :3].contiguous()},
               {"workspace": torch.zeros(16, dtype=torch.uint8, device=cuda_device)}):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in ({"q": d[0].float()}, {"lengths": d[7].float()}):
        with pytest.raises(TypeError):
            call(**kw)


def test_random_shapes(cuda_device):
    g = torch.Generator().manual_seed(77)

    def pick(values):
        return values[int(torch.randint(0, len(values), (1,), generator=g))]
    for i in range(25):
        kv = pick([1, 2, 3, 8])
        heads = kv * pick([1, 2, 4, 5, 16])
        sizes = [int(torch.randint(0, 20, (1,), generator=g)) for _ in range(pick([1, 2, 5]))]
        n = max(1, sum(sizes) + pick([0, 0, 3]))
        lens = torch.randint(0, pick([2, 100, 700]), (n,), generator=g).tolist()
        prefix = torch.randint(0, pick([2, 100, 3000]), (len(sizes),), generator=g).tolist()
        _run(_case(100 + i, sizes, lens, prefix, pick([4, 16, 17, 64]), heads, kv, pick([64, 128]),
                   pick([torch.bfloat16, torch.float16])), cuda_device)


@pytest.mark.parametrize("seed", range(40, 64))
def test_more_random_batches(cuda_device, seed):
    """Groups from one to many sequences, prompts and completions from nothing to several tiles."""
    g = torch.Generator().manual_seed(seed)
    pick = lambda *x: x[int(torch.randint(0, len(x), (1,), generator=g))]  # noqa: E731
    groups = [int(x) for x in torch.randint(0, pick(2, 9, 20), (pick(1, 3, 6),), generator=g)]
    n = max(1, sum(groups) + pick(0, 2))
    lengths = [int(x) for x in torch.randint(0, pick(2, 40, 300), (n,), generator=g)]
    prefix = [int(x) for x in torch.randint(0, pick(2, 100, 900), (len(groups),), generator=g)]
    kv = pick(1, 2, 5)
    _run(_case(seed, groups, lengths, prefix, pick(8, 13, 16, 32), kv * pick(1, 2, 4, 7, 8), kv, pick(64, 128),
               pick(torch.bfloat16, torch.float16)), cuda_device)


@pytest.mark.parametrize("block", [16, 32, 48, 64, 80, 128, 192])
@pytest.mark.parametrize("heads,kv", [(8, 2), (32, 1)])
def test_big_tiles_with_missing_and_repeated_pages(cuda_device, block, heads, kv):
    """More than sixteen rows a KV head and many tiles: pages that do not exist (their tile is copied row by
    row, between tiles of tensor copies), pages named twice, an end inside a page."""
    import tome_b200
    c = _case(block, [8], [33, 0, 200, 64, 1, 90, 5, 130], [3001], block, heads, kv, 128, torch.bfloat16)
    table = c["prefix_tables"]
    used = (3001 + block - 1) // block
    for i in {1, used // 3, used // 2, used - 1}:
        table[0, i] = -1 if i % 2 else c["k_pool"].shape[0]
    table[0, used // 4] = table[0, 0]
    c["tables"][2, 0] = table[0, 0]
    out, lse = tome_b200.shared_prefix_attention(*_dev(c, cuda_device), return_lse=True)
    with pytest.raises(tome_b200.TomeRuntimeError, match="block-table"):
        tome_b200.check_device_status(cuda_device)
    _compare(c, out, lse)


@pytest.mark.parametrize("block", [32, 64])
def test_what_lies_behind_a_big_prefix_is_not_read(cuda_device, block):
    c = _case(block, [12], [7] * 12, [block * 9 + 5], block, 8, 2, 64, torch.float16)
    want, want_lse = _run(c, cuda_device)
    last = int(c["prefix_tables"][0, 9])
    for pool in (c["k_pool"], c["v_pool"]):
        pool[last, :, 5:] = float("nan")
        named = torch.cat([c["prefix_tables"].reshape(-1), c["tables"].reshape(-1)]).long()
        rest = torch.ones(pool.shape[0], dtype=torch.bool)
        rest[named] = False
        pool[rest] = float("inf")
    import tome_b200
    got, got_lse = tome_b200.shared_prefix_attention(*_dev(c, cuda_device), return_lse=True, check=True)
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)


def test_as_many_sequences_and_groups_as_a_call_takes(cuda_device):
    import tome_b200
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 20, (2048,), generator=g).tolist()
    prefix = torch.randint(0, 70, (512,), generator=g).tolist()
    c = _case(31, [4] * 512, lens, prefix, 16, 8, 1, 64, torch.bfloat16)  # 32 rows a group: all prefixes big
    _run(c, cuda_device)
    more = dict(c, q=torch.cat([c["q"], c["q"][:1]]), tables=torch.cat([c["tables"], c["tables"][:1]]),
                lengths=torch.cat([c["lengths"], c["lengths"][:1]]))
    with pytest.raises(ValueError):
        tome_b200.shared_prefix_attention(*_dev(more, cuda_device))
