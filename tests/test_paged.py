"""Paged cache operators against plain 64-bit forms, on the CPU path and on the
HIP kernels."""

import math

import pytest
import torch

from luminaai_amd import ops

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _pool(pages, hkv, page, width, dev, dtype=torch.bfloat16, fill=math.nan):
    return torch.full((pages, hkv, page, width), fill, dtype=dtype, device=dev)


def _scene(lens, H, HKV, D, page, dev, spare=3, seed=0, layout="pages"):
    """Sequences over a shuffled pool that holds NaN wherever no live token
    lies, and their dense keys and values in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    W = ops.page_width(D)
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g)
    M = max(need + [1]) + 1
    table = torch.full((len(lens), M), total + 7, dtype=torch.int32)
    k, v = (_pool(total, HKV, page, W, "cpu") for _ in range(2))
    dense, at = [], 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]].int()
        at += need[b]
        kv = torch.randn(2, n, HKV, D, generator=g).bfloat16()
        for pool, new in ((k, kv[0]), (v, kv[1])):
            for t in range(n):
                pool[table[b, t // page].long(), :, t % page, :D] = new[t]
        dense.append(kv.double())
    q = (1.5 * torch.randn(len(lens), H, D, generator=g)).bfloat16()
    k, v = k.to(dev), v.to(dev)
    if layout == "tokens":        # [pages, page, kv_heads, width] underneath
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    elif layout == "layers":      # one layer of a pool over all layers
        k, v = (torch.stack([torch.full_like(t, math.nan), t])[1]
                for t in (k, v))
    return (q.to(dev), k, v, table.to(dev),
            torch.tensor(lens, dtype=torch.int32, device=dev), dense)


def _oracle(q, dense, D, live=None):
    """(o, tolerance) in 64 bits. The output is rounded once (2^-8 of its
    value); fp32 scores are off by at most D 2^-24 sum |q k| scale, which moves
    a probability by twice that and o by as much of max |v|; probabilities keep
    16 bits."""
    B, H, _ = q.shape
    outs, tols = [], []
    for b in range(B):
        k, v = dense[b]
        if live is not None:
            k, v = k[live[b]], v[live[b]]
        o = torch.zeros(H, D, dtype=torch.float64)
        tol = torch.zeros(H, D, dtype=torch.float64)
        if k.shape[0]:
            G = H // k.shape[1]
            for h in range(H):
                qh = q[b, h].double().cpu()
                s = k[:, h // G] @ qh / math.sqrt(D)
                e = (k[:, h // G].abs() @ qh.abs()).max() / math.sqrt(D)
                o[h] = s.softmax(0) @ v[:, h // G]
                tol[h] = o[h].abs() * 2 ** -8 + v[:, h // G].abs().max() * (
                    2 ** -15 + 2 * (D + 4) * 2 ** -24 * e)
        outs.append(o)
        tols.append(tol)
    return torch.stack(outs), torch.stack(tols)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("H,HKV,D", [(4, 4, 8), (2, 1, 15), (8, 4, 64),
                                     (8, 8, 80), (8, 2, 96), (32, 8, 128),
                                     (12, 4, 159), (4, 4, 192), (34, 2, 40)])
@pytest.mark.parametrize("page", [16, 64])
def test_paged_attention(dev, H, HKV, D, page):
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 63, 130, 300]
    q, k, v, table, n, dense = _scene(lens, H, HKV, D, page, dev)
    o = ops.paged_attention(q, k, v, table, n)
    assert o.dtype == q.dtype and o.shape == q.shape
    ref, tol = _oracle(q, dense, D)
    assert ((o.double().cpu() - ref).abs() <= tol).all()
    assert (o[0] == 0).all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("layout", ["tokens", "layers"])
def test_paged_attention_layouts(dev, layout):
    """Pools of other strides, and q as a view of the fused projection."""
    q, k, v, table, n, dense = _scene([45, 3, 200], 12, 4, 159, 32, dev,
                                      layout=layout)
    wide = torch.zeros(3, 12 + 8, 159, dtype=q.dtype, device=dev)
    wide[:, :12] = q
    o = ops.paged_attention(wide[:, :12], k, v, table, n, scale=159 ** -0.5)
    ref, tol = _oracle(q, dense, 159)
    assert ((o.double().cpu() - ref).abs() <= tol).all()
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)     # channels apart
    assert torch.equal(ops.paged_attention(qt, k, v, table, n), o)


@pytest.mark.parametrize("dev", DEVS)
def test_paged_attention_bad_pages_and_lengths(dev):
    """Tokens of page numbers outside the pool are left out; lengths are cut to
    the table."""
    page, D = 16, 64
    q, k, v, table, n, dense = _scene([100, 40, 64, 20], 4, 2, D, page, dev)
    live = [torch.ones(x, dtype=torch.bool) for x in (100, 40, 64, 20)]
    table[0, 2] = -1
    table[0, 5] = 2 ** 31 - 1
    live[0][32:48] = False
    live[0][80:96] = False
    table[1, :] = 10 ** 6
    live[1][:] = False
    n[3] = -5
    live[3][:] = False
    o = ops.paged_attention(q, k, v, table, n)
    ref, tol = _oracle(q, dense, D, live)
    assert ((o.double().cpu() - ref).abs() <= tol).all()
    assert (o[1] == 0).all() and (o[3] == 0).all()
    # past the row: 64 tokens fill four pages
    o2 = ops.paged_attention(q[2:3], k, v, table[2:3, :4],
                             torch.tensor([10 ** 9], dtype=torch.int32,
                                          device=dev))
    assert torch.equal(o2, o[2:3])


@pytest.mark.parametrize("dev", DEVS)
def test_paged_attention_large_scores(dev):
    """Scores far apart: the running maximum moves late and by much."""
    q, k, v, table, n, dense = _scene([700], 2, 1, 64, 16, dev, seed=3)
    for i, t in enumerate((5, 300, 650)):
        page = table[0, t // 16].long()
        k[page, :, t % 16, :64] = q[0, 0] * (2.0 ** (i + 1))
        dense[0][0, t] = k[page, :, t % 16, :64].double().cpu()
    o = ops.paged_attention(q, k, v, table, n)
    ref, tol = _oracle(q, dense, 64)
    assert ((o.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("D", [40, 64, 159])
def test_scores_of_minus_infinity(dev, D):
    """Such tokens have no weight, also where a chunk holds nothing else; a
    sequence of nothing else has no softmax, unlike one without tokens."""
    lens = [20, 20, 3000, 3000, 0, 1, 16]
    q, k, v, table, n, dense = _scene(lens, 4, 2, D, 16, dev)
    q = q.abs() + 0.25
    live = [torch.ones(x, dtype=torch.bool) for x in lens]
    live[0][:] = live[3][:] = live[5][:] = False        # all of them
    live[1][[0, 1, 2, 5, 19]] = False
    live[2][:2500] = False                              # whole chunks
    for b, keep in enumerate(live):
        for t in (~keep).nonzero()[:, 0].tolist():
            k[table[b, t // 16].long(), :, t % 16, :D] = -math.inf
    o = ops.paged_attention(q, k, v, table, n)
    assert o[[0, 3, 5]].isnan().all()
    ref, tol = _oracle(q, dense, D, live)
    rest = [1, 2, 4, 6]
    assert ((o.double().cpu() - ref).abs() <= tol)[rest].all()
    assert (o[4] == 0).all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
@pytest.mark.parametrize("D,page", [(159, 16), (64, 128), (15, 32)])
def test_paged_append(dev, dtype, D, page):
    HKV, W = 3, ops.page_width(D)
    fused = torch.randn(40, 2 * HKV * D + 1, device=dev).to(dtype)
    k = fused[:, :HKV * D].view(40, HKV, D)
    v = fused[:, HKV * D:2 * HKV * D].view(40, HKV, D)
    kp, vp = (_pool(9, HKV, page, W, dev, dtype, 7.0) for _ in range(2))
    table = torch.tensor([[4, 2, 8], [0, 5, 1], [3, -1, 99]],
                         dtype=torch.int32, device=dev)
    ids = torch.tensor([0] * 20 + [1] * 10 + [2] * 6 + [3, -1, 1, 0],
                       dtype=torch.int32, device=dev)
    pos = list(range(page - 10, page + 10)) + list(range(2 * page, 2 * page
                                                         + 10))
    pos += [0, 1, page, page + 1, 2 * page, 3 * page]   # seq 2: pages 3, -, -
    pos += [0, 0, -1, 3 * page]                         # places that are not
    pos = torch.tensor(pos, dtype=torch.int32, device=dev)
    want = [t.clone() for t in (kp, vp)]
    for t in range(40):
        b, p = int(ids[t]), int(pos[t])
        if not 0 <= b < 3 or not 0 <= p < 3 * page:
            continue
        pg = int(table[b, p // page])
        if not 0 <= pg < 9:
            continue
        for pool, new in zip(want, (k, v)):
            pool[pg, :, p % page, :D] = new[t]
            pool[pg, :, p % page, D:] = 0
    ops.paged_kv_append(k, v, kp, vp, table, pos, ids)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


@pytest.mark.parametrize("dev", DEVS)
def test_paged_append_one_token_each(dev):
    """Without seq_ids token t belongs to sequence t; tokens without channels
    beside each other are taken too."""
    kp, vp = (_pool(4, 2, 16, 8, dev, fill=0.0) for _ in range(2))
    k = torch.randn(2, 8, 3, device=dev).bfloat16().permute(2, 0, 1)
    table = torch.tensor([[1], [3], [0]], dtype=torch.int32, device=dev)
    pos = torch.tensor([5, 0, 15], dtype=torch.int32, device=dev)
    ops.paged_kv_append(k, -k, kp, vp, table, pos)
    for t, (pg, row) in enumerate([(1, 5), (3, 0), (0, 15)]):
        assert torch.equal(kp[pg, :, row], k[t])
        assert torch.equal(vp[pg, :, row], -k[t])
    assert int((kp != 0).any(-1).sum()) == 6
    empty = k[:0]
    ops.paged_kv_append(empty, empty, kp, vp, table[:0], pos[:0])


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype,tail", [(torch.bfloat16, (2, 16, 160)),
                                        (torch.float32, (1, 32, 200)),
                                        (torch.int8, (37,)),
                                        (torch.bfloat16, (4, 128, 128))])
@pytest.mark.parametrize("pairs", [1, 300])
def test_copy_pages(dev, dtype, tail, pairs):
    P = 2 * pairs + 5
    pool = (torch.randn(3, P, *tail, device=dev) * 50).to(dtype)
    other = (torch.randn(2, P + 1, 5, device=dev) * 50).to(dtype)
    order = torch.randperm(P, generator=torch.Generator().manual_seed(1))
    src, dst = order[:pairs].tolist(), order[pairs:2 * pairs].tolist()
    src[-1] = src[0]                              # one source, two forks
    want = [pool.clone(), pool.clone() + 1, other.clone()]
    pools = [w.clone() for w in want]
    for w in want:
        for a, b in zip(src, dst):
            w[:, b] = w[:, a]
    ops.copy_pages(pools, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    # layers apart from each other, pages in another order
    big = torch.zeros(P, 6, *tail, dtype=dtype, device=dev)
    view = big[:, ::2].transpose(0, 1)
    view.copy_(pool)
    ops.copy_pages([view], src, dst)
    assert torch.equal(view, want[0]) and (big[:, 1::2] == 0).all()
    ops.copy_pages([pool], [], [])


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("HKV,D,dtype", [(4, 159, torch.bfloat16),
                                         (8, 128, torch.bfloat16),
                                         (1, 20, torch.float32)])
@pytest.mark.parametrize("T", [2047, 2051, 4099])
def test_append_of_many_tokens(dev, HKV, D, dtype, T):
    """On both sides of the sizes that a workgroup's share depends on."""
    g = torch.Generator().manual_seed(T)
    kv = torch.randn(2, T, HKV, D, generator=g).to(dtype).to(dev)
    page, W = 64, ops.page_width(D)
    n = -(-T // page) + 1
    k, v = (torch.full((n, HKV, page, W), 7.0, dtype=dtype, device=dev)
            for _ in range(2))
    table = torch.randperm(n, generator=g).int()
    pos = torch.arange(T, dtype=torch.int32)
    pos[5::97] = -1
    ops.paged_kv_append(kv[0], kv[1], k, v, table[None].to(dev), pos.to(dev),
                        torch.zeros(T, dtype=torch.int32, device=dev))
    live = pos >= 0
    for new, pool in zip(kv, (k, v)):
        seq = pool.cpu()[table.long()].transpose(1, 2).reshape(-1, HKV, W)
        assert torch.equal(seq[:T][live][..., :D], new.cpu()[live])
        assert (seq[:T][live][..., D:] == 0).all()
        assert (seq[:T][~live] == 7).all() and (seq[T:] == 7).all()


@pytest.mark.parametrize("dev", DEVS)
def test_append_attend_fork(dev):
    """A sequence is written token by token, forked inside a page, and both
    continue: each attends to what it wrote."""
    H, HKV, D, page = 6, 2, 40, 16
    g = torch.Generator().manual_seed(5)
    pools = [_pool(8, HKV, page, 40, dev)[None] for _ in range(2)]
    table = torch.tensor([[6, 1, 3], [6, 4, 0]], dtype=torch.int32, device=dev)
    new = torch.randn(2, 2, 40, HKV, D, generator=g).bfloat16().to(dev)
    new[:, 1, :21] = new[:, 0, :21]               # the shared prompt
    kp, vp = pools[0][0], pools[1][0]
    pos = torch.arange(21, dtype=torch.int32, device=dev)
    ops.paged_kv_append(new[0, 0, :21], new[1, 0, :21], kp, vp, table, pos,
                        torch.zeros_like(pos))
    ops.copy_pages(pools, [1], [4])
    for t in range(21, 40):
        at = torch.full((2,), t, dtype=torch.int32, device=dev)
        ops.paged_kv_append(new[0, :, t], new[1, :, t], kp, vp, table, at)
        if t in (21, 31, 32, 39):
            q = torch.randn(2, H, D, generator=g).bfloat16().to(dev)
            o = ops.paged_attention(q, kp, vp, table, at + 1)
            dense = [new[:, b, :t + 1].double().cpu() for b in range(2)]
            ref, tol = _oracle(q, dense, D)
            assert ((o.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dev", DEVS)
def test_writes_are_seen_by_autograd(dev):
    """A pool that a backward pass needs may not have been written since."""
    k = torch.zeros(2, 6, 1, 16, 8, device=dev)
    v = torch.zeros_like(k)
    table = torch.zeros(1, 2, dtype=torch.int32, device=dev)
    new = torch.ones(1, 1, 8, device=dev)
    pos = torch.zeros(1, dtype=torch.int32, device=dev)
    x = torch.ones(8, device=dev, requires_grad=True)
    for write in (lambda: ops.paged_kv_append(new, new, k[0], v[0], table, pos),
                  lambda: ops.copy_pages([k, v], [0], [1])):
        for pool in (k, v):
            before = pool._version
            loss = (pool * x).sum()
            write()
            assert pool._version > before
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                loss.backward()
    # what was made in inference mode has no versions
    with torch.inference_mode():
        k, v = k.clone(), v.clone()
        ops.paged_kv_append(new, new, k[0], v[0], table, pos)
        ops.copy_pages([k, v], [0], [1])
        # one row of 8 in page 0 and its copy in page 1
        assert float(k.sum()) == float(v.sum()) == 16


@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    q, k, v, table, n, _ = _scene([20, 5], 4, 2, 64, 16, dev)

    def refuse(err, match, fn=ops.paged_attention, args=(), **kw):
        with pytest.raises(err, match=match):
            fn(*args, **kw)

    A = (q, k, v, table, n)

    def swap(i, x):
        return A[:i] + (x,) + A[i + 1:]

    refuse(ValueError, "batch, heads", args=swap(0, q[0]))
    refuse(ValueError, "multiple of kv_heads", args=swap(0, q[:, :3]))
    refuse(ValueError, "wide", args=swap(0, q[..., :50]))
    refuse(ValueError, "1 to 192", args=swap(0, q.repeat(1, 1, 4)))
    refuse(TypeError, "k_pages is", args=swap(1, k.float())[:2]
           + (v.float(), table, n))
    refuse(ValueError, "one shape", args=swap(2, v[:, :1]))
    refuse(ValueError, "power of two",
           args=(q, k[:, :, :12], v[:, :, :12], table, n))
    refuse(TypeError, "block_table must be int32", args=swap(3, table.long()))
    refuse(TypeError, "seq_lens must be int32", args=swap(4, n.long()))
    refuse(ValueError, "2-dimensional", args=swap(3, table[0]))
    refuse(ValueError, "each of the 2 sequences", args=swap(4, n[:1]))
    refuse(RuntimeError, "no gradient",
           args=swap(0, q.clone().requires_grad_(True)))
    kn = k.new_zeros(2, 2, 64)
    P = torch.zeros(2, dtype=torch.int32, device=dev)
    app = ops.paged_kv_append
    refuse(ValueError, "tokens, kv_heads", app, (kn[0], kn[0], k, v, table, P))
    refuse(TypeError, "v is", app, (kn, kn.float(), k, v, table, P))
    refuse(ValueError, "heads, not 1", app, (kn[:, :1], kn[:, :1], k, v, table,
                                             P))
    refuse(ValueError, "positions has 1", app, (kn, kn, k, v, table, P[:1]))
    refuse(ValueError, "one token for each", app, (kn, kn, k, v, table[:1], P))
    refuse(ValueError, "seq_ids has", app, (kn, kn, k, v, table, P, P[:1]))
    pool = k[None]
    cp = ops.copy_pages
    refuse(ValueError, "src names", cp, ([pool], [0, 1], [2]))
    refuse(ValueError, "written twice", cp, ([pool], [0, 1], [2, 2]))
    refuse(ValueError, "both read and written", cp, ([pool], [0, 1], [1, 2]))
    refuse(ValueError, "page numbers", cp, ([pool], [0], [k.shape[0]]))
    refuse(ValueError, "page numbers", cp, ([pool], [-1], [0]))
    refuse(ValueError, "no pool", cp, ([], [0], [1]))
    refuse(ValueError, "layers, pages", cp, ([pool[0, 0, 0]], [0], [1]))
    refuse(ValueError, "contiguous", cp, ([pool.transpose(2, 3)], [0], [1]))
    # memory that several pages share
    same = k[:1].expand(k.shape)
    refuse(ValueError, "overlaps", cp, ([same[None]], [0], [1]))
    refuse(ValueError, "overlaps", cp, ([pool.expand(2, *k.shape)], [0], [1]))
    refuse(ValueError, "overlaps", app, (kn, kn, same, v, table, P))
    refuse(ValueError, "overlaps", app, (kn, kn, k, k, table, P))
    refuse(RuntimeError, "no gradient",
           args=swap(1, k.clone().requires_grad_(True)))
    for scale in (math.inf, math.nan, 1e31):
        refuse(ValueError, "scale", args=(*A, scale))


@pytest.mark.parametrize("dev", DEVS)
def test_huge_scores(dev):
    """Scores near the end of the range on either side, all of one sign: the
    mean of the values, not zeros."""
    q, k, v, table, n, _ = _scene([20, 300], 4, 2, 64, 16, dev)
    for sign in (-1, 1):
        q.fill_(2.0 ** 60)
        k.fill_(sign * 2.0 ** 60)
        v.fill_(1.5)
        o = ops.paged_attention(q, k, v, table, n)
        assert torch.equal(o, torch.full_like(o, 1.5))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("lens", [
    [(37 * b) % 200 for b in range(130)], [0] * 64 + [900],
    [900] + [0] * 70 + [1, 300], [128, 129, 256, 257, 1023, 1024, 1025],
    [2, 0, 1] * 350 + [700, 3]])
def test_rows_and_widths(dev, lens):
    """More rows than lanes, empty ones among them; however wide the table is,
    the result is the same."""
    q, k, v, table, n, dense = _scene(lens, 4, 2, 64, 16, dev)
    o, tol = _oracle(q, dense, 64)
    wide = torch.nn.functional.pad(table, (0, 3000 - table.shape[1]), value=-1)
    for t in (table, wide):
        got = ops.paged_attention(q, k, v, t, n).double().cpu()
        assert ((got - o).abs() <= tol).all()


@pytest.mark.parametrize("dev", DEVS)
def test_columns_of_one(dev):
    """A table or lengths of one entry have no order that could be wrong."""
    q, k, v, table, n, _ = _scene([9], 4, 2, 64, 16, dev)
    t = torch.stack([table, table], -1)[:, :1, 0]
    m = torch.stack([n, n], -1)[:, 0]
    assert torch.equal(ops.paged_attention(q, k, v, t, m),
                       ops.paged_attention(q, k, v, table, n))


@pytest.mark.gpu
def test_gpu_refusals():
    q, k, v, table, n, _ = _scene([20, 5], 4, 2, 64, 16, "cuda")
    with pytest.raises(TypeError, match="bf16"):
        ops.paged_attention(q.float(), k.float(), v.float(), table, n)
    with pytest.raises(ValueError, match="block_table is on cpu"):
        ops.paged_attention(q, k, v, table.cpu(), n)
    with pytest.raises(ValueError, match="k_pages is on cpu"):
        ops.paged_attention(q, k.cpu(), v, table, n)
    for rows, cols in ((1, 2 ** 25), (2 ** 10, 2 ** 18)):
        far = table.new_zeros(1, cols).expand(rows, cols)
        with pytest.raises(ValueError, match="2\\^29|2\\^31"):
            ops.paged_attention(q[:1].expand(rows, 4, 64), k, v, far,
                                n[:1].repeat(rows))
    with pytest.raises(ValueError, match="16-byte aligned"):
        odd = torch.zeros(k.numel() + 1, dtype=k.dtype,
                          device="cuda")[1:].view(k.shape)
        ops.paged_attention(q, odd, odd, table, n)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements, its last pages in use."""
    HKV, page, W = 8, 128, 128
    P = 2 ** 32 // (HKV * page * W) + 40
    q, k, v, table, n, dense = _scene([1500, 77], 16, HKV, W, page, "cuda")
    big = [torch.empty(P, HKV, page, W, dtype=torch.bfloat16, device="cuda")
           for _ in range(2)]
    small = k.shape[0]
    for pool, x in zip(big, (k, v)):
        pool[P - small:] = x
    far = torch.where(table < small, table + (P - small), table)
    o = ops.paged_attention(q, big[0], big[1], far, n)
    assert torch.equal(o, ops.paged_attention(q, k, v, table, n))
    src = int(far[1, 0])
    ops.copy_pages([t[None] for t in big], [src], [P - small - 1])
    assert torch.equal(big[0][src].view(torch.int16),
                       big[0][P - small - 1].view(torch.int16))
    at = torch.tensor([3, 5], dtype=torch.int32, device="cuda")
    kn = torch.randn(2, HKV, W, device="cuda").bfloat16()
    ops.paged_kv_append(kn, kn, big[0], big[1], far, at)
    assert torch.equal(big[1][src, :, 5], kn[1])


@pytest.mark.gpu
def test_capture_and_replay():
    """A captured step follows tables and lengths that change between its
    replays, while the same calls run eagerly beside it."""
    H, HKV, D, page = 12, 4, 159, 16
    q, k, v, table, n, _ = _scene([700, 30, 1], H, HKV, D, page, "cuda")
    kn = torch.randn(3, HKV, D, device="cuda").bfloat16()
    table = torch.arange(3 * table.shape[1], dtype=torch.int32, device="cuda"
                         ).view(3, -1) % k.shape[0]
    k.nan_to_num_(0.5)
    v.nan_to_num_(0.25)

    def step():
        ops.paged_kv_append(kn, kn, k, v, table, n - 1)
        return ops.paged_attention(q, k, v, table, n)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        n.copy_(torch.tensor([703 - 97 * i, 30 + i, 0 if i == 2 else 1 + i],
                             dtype=torch.int32))
        table.copy_(table.roll(1, 1))
        q.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_other_stream():
    q, k, v, table, n, dense = _scene([900, 513], 8, 8, 128, 64, "cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o = ops.paged_attention(q, k, v, table, n)
    s.synchronize()
    ref, tol = _oracle(q, dense, 128)
    assert ((o.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls under way on two streams, with planned chunks and without."""
    sides = []
    for lens in ([3000, 17, 900], [40, 0, 300] * 60):
        q, k, v, table, n, _ = _scene(lens, 8, 2, 64, 16, "cuda")
        sides.append((q, k, v, table, n))
    ref = [ops.paged_attention(*a) for a in sides]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    got = [[], []]
    for _ in range(20):
        for out, st, a in zip(got, streams, sides):
            with torch.cuda.stream(st):
                out.append(ops.paged_attention(*a))
    torch.cuda.synchronize()
    for outs, r in zip(got, ref):
        assert all(torch.equal(o, r) for o in outs)


@pytest.mark.gpu
def test_planned_chunks_in_a_graph():
    """More rows than a workgroup looks through; lengths change between
    replays."""
    lens = [40, 0, 300] * 60
    q, k, v, table, n, _ = _scene(lens, 8, 2, 64, 16, "cuda")
    with torch.no_grad():
        ops.paged_attention(q, k, v, table, n)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_attention(q, k, v, table, n)
        for step in range(4):
            n.copy_(torch.tensor([max(0, x - 7 * step) for x in lens]).int())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out.clone(), ops.paged_attention(q, k, v, table,
                                                                n))
