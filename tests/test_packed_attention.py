"""Packed causal attention against plain 64-bit forms, on the CPU path and on the
HIP kernels, with gradients."""

import math

import pytest
import torch
import torch.utils.checkpoint

from luminaai_amd import ops

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HALF = 2.0 ** -8              # one rounding to bf16


def _cu(lens, dev):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=dev)


def _inputs(lens, tail, H, HKV, D, dev, seed=0, std=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + tail
    qkv = torch.randn(T, (H + 2 * HKV) * D, generator=g).to(dtype).to(dev)
    q, k, v = qkv.split([H * D, HKV * D, HKV * D], dim=1)
    go = torch.randn(T, H, D, generator=g).to(dtype).to(dev)
    return (q.view(T, H, D) * std, k.view(T, HKV, D), v.view(T, HKV, D), go)


def _oracle(q, k, v, go, lens, scale):
    """Values and tolerances in 64 bits. Each bf16 rounding is off by 2^-8 of
    its value: the results', P's and dS's as operands, o's inside delta. fp32
    scores are off by (D + 4) 2^-24 sum |q k| scale, a probability by twice
    that relative."""
    q, k, v, go = (t.detach().double().cpu() for t in (q, k, v, go))
    T, H, D = q.shape
    G = H // k.shape[1]
    val = [torch.zeros_like(t) for t in (q, q, k, v)]
    tol = [torch.zeros_like(t) for t in (q, q, k, v)]
    at = 0
    for n in lens:
        sl = slice(at, at + n)
        at += n
        if not n:
            continue
        tri = torch.ones(n, n, dtype=torch.bool).tril()
        for h in range(H):
            Q, K, V, dO = q[sl, h], k[sl, h // G], v[sl, h // G], go[sl, h]
            S = (Q @ K.t()) * scale
            eps = 2 * (D + 4) * 2.0 ** -24 * float(
                (Q.abs() @ K.abs().t()).max()) * scale
            P = S.masked_fill(~tri, -math.inf).softmax(-1)
            O = P @ V
            dO_tol = HALF * O.abs() + (HALF + 2 * eps) * (P @ V.abs())
            val[0][sl, h], tol[0][sl, h] = O, dO_tol
            dP = dO @ V.t()
            dS = P * (dP - (dO * O).sum(-1, keepdim=True))
            e = (HALF + 2 * eps) * dS.abs() + P * (
                (dO.abs() * dO_tol).sum(-1, keepdim=True)
                + 2 * D * 2.0 ** -24 * (dO.abs() @ V.abs().t()))
            val[1][sl, h] = dS @ K * scale
            tol[1][sl, h] = e @ K.abs() * scale
            val[2][sl, h // G] += dS.t() @ Q * scale
            tol[2][sl, h // G] += e.t() @ Q.abs() * scale
            val[3][sl, h // G] += P.t() @ dO
            tol[3][sl, h // G] += (HALF + 2 * eps) * (P.t() @ dO.abs())
    for i in (1, 2, 3):
        tol[i] += HALF * val[i].abs() + 2.0 ** -20 * tol[i]
    return val, tol


def _check(got, val, tol):
    for name, x, y, t in zip(("o", "dq", "dk", "dv"), got, val, tol):
        off = (x.detach().double().cpu() - y).abs() - t
        assert x.shape == y.shape and (off <= 2.0 ** -126).all(), (
            name, float(off.max()))


def _run(q, k, v, go, cu, scale=None):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = ops.flash_attention_packed(*leaves, cu, scale)
    return (o, *torch.autograd.grad(o, leaves, go))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("H,HKV,D", [(2, 1, 5), (4, 4, 8), (4, 2, 15),
                                     (8, 4, 64), (2, 2, 80), (8, 2, 96),
                                     (8, 2, 128), (6, 2, 159), (3, 1, 160),
                                     (4, 4, 192), (16, 8, 32)])
def test_packed_attention(dev, H, HKV, D):
    lens = [1, 0, 31, 32, 33, 64, 65, 129, 300, 2]
    q, k, v, go = _inputs(lens, 7, H, HKV, D, dev)
    got = _run(q, k, v, go, _cu(lens, dev))
    val, tol = _oracle(q, k, v, go, lens, D ** -0.5)
    _check(got, val, tol)
    for t in got:
        assert (t[sum(lens):] == 0).all()
    with torch.no_grad():
        assert torch.equal(ops.flash_attention_packed(q, k, v,
                                                      _cu(lens, dev)), got[0])


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("H,HKV,D", [(2, 1, 5), (8, 4, 64), (2, 2, 80),
                                     (8, 2, 128), (6, 2, 159), (4, 4, 192)])
def test_few_tokens(dev, H, HKV, D):
    lens = [1, 0, 33, 129, 300]
    q, k, v, go = _inputs(lens, 7, H, HKV, D, dev, seed=1)
    _check(_run(q, k, v, go, _cu(lens, dev)),
           *_oracle(q, k, v, go, lens, D ** -0.5))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("H,HKV,D", [(8, 1, 15), (8, 4, 64), (8, 8, 80),
                                     (8, 2, 128), (9, 3, 159), (8, 8, 192)])
def test_more_tokens(dev, H, HKV, D):
    lens = [700, 1, 0, 400]
    q, k, v, go = _inputs(lens, 7, H, HKV, D, dev, seed=2)
    _check(_run(q, k, v, go, _cu(lens, dev)),
           *_oracle(q, k, v, go, lens, D ** -0.5))


@pytest.mark.gpu
def test_few_roundings_of_a_small_call():
    """P and dS of a small call enter their products with 16 bits, so the
    gradients are little further off than their own rounding: a half of what
    a second rounding of the same size would add to its square."""
    lens = [43, 9]
    q, k, v, go = _inputs(lens, 5, 2, 1, 64, "cuda")
    got = _run(q, k, v, go, _cu(lens, "cuda"))
    val, _ = _oracle(q, k, v, go, lens, 0.125)
    for x, y in list(zip(got, val))[1:]:
        alone = (y.bfloat16().double() - y).norm()
        assert (x.double().cpu() - y).norm() <= 1.5 ** 0.5 * alone


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("lens,tail", [([], 5), ([0, 0], 3), ([1], 0),
                                       ([257], 0), ([1] * 150, 1),
                                       ([700, 3, 520], 300)])
def test_borders(dev, lens, tail):
    q, k, v, go = _inputs(lens, tail, 2, 1, 64, dev, seed=len(lens))
    got = _run(q, k, v, go, _cu(lens, dev))
    val, tol = _oracle(q, k, v, go, lens, 64 ** -0.5)
    _check(got, val, tol)


@pytest.mark.parametrize("dev", DEVS)
def test_no_tokens(dev):
    q, k, v, go = _inputs([], 0, 2, 1, 64, dev)
    got = _run(q, k, v, go, _cu([0], dev))
    assert [t.shape[0] for t in got] == [0] * 4


@pytest.mark.parametrize("dev", DEVS)
def test_strides_and_scale(dev):
    """Channels, heads and tokens in other orders; a broadcast gradient; a scale
    of the caller's."""
    lens = [70, 40]
    q, k, v, go = _inputs(lens, 0, 4, 2, 40, dev, seed=4)
    cu = _cu(lens, dev)
    val, tol = _oracle(q, k, v, go, lens, 0.3)
    ref = _run(q, k, v, go, cu, 0.3)
    _check(ref, val, tol)
    q2 = q.permute(1, 0, 2).contiguous().permute(1, 0, 2)    # heads first
    k2 = k.permute(2, 1, 0).contiguous().permute(2, 1, 0)    # channels first
    for a, b in zip(_run(q2, k2, v.flip(0).flip(0), go, cu, 0.3), ref):
        assert torch.equal(a, b)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    ops.flash_attention_packed(*leaves, cu, 0.3).sum().backward()
    one = _run(q, k, v, torch.ones_like(go), cu, 0.3)
    for a, b in zip(leaves, one[1:]):
        assert torch.equal(a.grad, b)


@pytest.mark.parametrize("dev", DEVS)
def test_keys_shared_by_broadcast(dev):
    """k and v expanded over the heads of a group, and one tensor for both: the
    gradients of every use add up."""
    lens = [50, 21]
    q, k, _, go = _inputs(lens, 0, 4, 1, 64, dev, seed=9)
    kv = k.detach().requires_grad_(True)
    wide = kv.expand(-1, 4, -1)
    o = ops.flash_attention_packed(q, wide, wide, _cu(lens, dev))
    g, = torch.autograd.grad(o, kv, go)
    _, _, dk, dv = _run(q, k, k, go, _cu(lens, dev))
    val, tol = _oracle(q, k, k, go, lens, 64 ** -0.5)
    # four roundings of the heads' parts and those of their sum
    want = val[2] + val[3]
    room = 4 * (tol[2] + tol[3]) + 8 * HALF * (val[2].abs() + val[3].abs())
    assert ((g.double().cpu() - want).abs() <= room).all()
    assert torch.equal(o, ops.flash_attention_packed(q, k, k, _cu(lens, dev)))
    assert ((dk + dv).double().cpu() - want).abs().le(room).all()


@pytest.mark.parametrize("dev", DEVS)
def test_late_maximum(dev):
    """Scores that rise by far more than the lazy maximum's 2^8 late in a row,
    and rows whose first keys hold all the weight."""
    lens = [400]
    q, k, v, go = _inputs(lens, 0, 2, 1, 64, dev, seed=6)
    k, q = k.clone(), q.clone()
    for i, t in enumerate((3, 130, 131, 390)):
        k[t] = q[399, 0] * (1.5 ** i)
    q[200:, 1] = q[200:, 1] * 6
    got = _run(q, k, v, go, _cu(lens, dev))
    val, tol = _oracle(q, k, v, go, lens, 64 ** -0.5)
    _check(got, val, tol)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [40, 900])
def test_scores_of_minus_infinity(dev, D, n):
    """A query with nothing else has no softmax; for the others such keys have
    no weight; other sequences do not notice, nor do their gradients."""
    lens = [20, n, 30]
    q, k, v, go = _inputs(lens, 0, 4, 2, D, dev, seed=n)
    q = q.abs() + 0.25
    k = k.clone()
    cu = _cu(lens, dev)
    plain = _run(q, k, v, go, cu)
    dead = n // 2
    k[:20] = -math.inf
    k[20:20 + dead] = -math.inf
    got = _run(q, k, v, go, cu)
    assert got[0][:20 + dead].isnan().all()
    for a, b in zip(plain, got):
        assert torch.equal(a[20 + n:], b[20 + n:])
    # the oracle on the keys that are left, which sit behind the dead ones: each
    # query sees those up to its own
    left = slice(20 + dead, 20 + n)
    val, tol = _oracle(q[left], k[left], v[left], go[left], [n - dead],
                       D ** -0.5)
    _check([got[0][left]], val[:1], tol[:1])


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("H,HKV,D,lens", [
    (8, 4, 64, [50] * 13), (8, 4, 64, [600, 700]), (8, 4, 64, [8, 900, 1] * 2),
    (2, 1, 96, [10] * 70), (4, 2, 64, [10] * 70), (2, 2, 192, [130] * 5),
    (2, 2, 192, [20] * 40), (2, 1, 53, [33] * 62), (2, 1, 53, [33] * 63)])
def test_few_long_and_many_short(dev, H, HKV, D, lens):
    """Both arrangements of the forward's waves, on either side of the sizes
    that choose between them."""
    q, k, v, go = _inputs(lens, 1, H, HKV, D, dev, seed=len(lens))
    val, tol = _oracle(q, k, v, go, lens, D ** -0.5)
    _check(_run(q, k, v, go, _cu(lens, dev)), val, tol)


@pytest.mark.parametrize("dev", DEVS)
def test_gradient_against_differences(dev):
    """sum(o go) at two points h apart along a direction, in 64 bits from the
    returned o, against the gradient's product with it. The difference is off by
    o's roundings, which the oracle's tolerance bounds, and by h^2 / 6 times
    the third derivative, here under 1 % of the bound."""
    lens = [37, 12]
    D, h = 32, 2.0 ** -3
    q, k, v, go = _inputs(lens, 0, 2, 1, D, dev, seed=8)
    cu = _cu(lens, dev)
    grads = _run(q, k, v, go, cu)[1:]
    gen = torch.Generator().manual_seed(1)
    for i in range(3):
        base = [q, k, v]
        d = (torch.randint(0, 2, base[i].shape, generator=gen) * 2.0 - 1).to(
            dev) * base[i].float().abs().clamp(2.0 ** -4, 1)
        pts = []
        for s in (h, -h):
            pts.append((base[i].float() + s * d).bfloat16())
        step = (pts[0].double() - pts[1].double())
        f, room = [], 0.0
        for p in pts:
            a = list(base)
            a[i] = p
            o = ops.flash_attention_packed(*a, cu)
            f.append(float((o.double() * go.double()).sum()))
            val, tol = _oracle(*a, go, lens, D ** -0.5)
            room += float((tol[0] * go.double().cpu().abs()).square().sum()
                          .sqrt()) * 4
        mid = list(base)
        mid[i] = ((pts[0].double() + pts[1].double()) / 2).bfloat16()
        slope = float((grads[i].double() * step).sum())
        _, tol = _oracle(*base, go, lens, D ** -0.5)
        room += float((tol[i + 1] * step.cpu().abs()).square().sum().sqrt()) * 4
        # the third derivative along a step of relative size h: h^2 of the
        # change, and the midpoint's rounding: 2^-8 of it
        room += (h * h + 2 * HALF) * float(
            (grads[i].double() * step).abs().sum())
        assert abs((f[0] - f[1]) - slope) <= room


def test_gradcheck_of_the_cpu_form():
    q, k, v, _ = _inputs([5, 0, 3], 1, 4, 2, 3, "cpu", dtype=torch.float64)
    cu = _cu([5, 0, 3], "cpu")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    assert torch.autograd.gradcheck(
        lambda a, b, c: ops.flash_attention_packed(a, b, c, cu), leaves)


@pytest.mark.parametrize("dev", DEVS)
def test_same_each_time(dev):
    lens = [333, 95]
    q, k, v, go = _inputs(lens, 0, 4, 2, 128, dev)
    cu = _cu(lens, dev)
    first = _run(q, k, v, go, cu)
    for _ in range(2):
        for a, b in zip(first, _run(q, k, v, go, cu)):
            assert torch.equal(a, b)


def test_positions():
    cu = _cu([3, 0, 2], "cpu")
    assert ops.packed_positions(cu, 7).tolist() == [[0, 1, 2, 0, 1, 0, 1]]


@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    q, k, v, _ = _inputs([6], 0, 4, 2, 64, dev)
    cu = _cu([6], dev)
    f = ops.flash_attention_packed
    for err, match, args in [
            (ValueError, "tokens, heads", (q[0], k, v, cu)),
            (ValueError, "tokens, heads", (q, k, v[:, :1], cu)),
            (ValueError, "same tokens", (q, k[:5], v[:5], cu)),
            (ValueError, "same tokens", (q, k[..., :8], v[..., :8], cu)),
            (ValueError, "multiple of kv_heads", (q[:, :3], k, v, cu)),
            (ValueError, "1 to 192", (q.repeat(1, 1, 4), k.repeat(1, 1, 4),
                                      v.repeat(1, 1, 4), cu)),
            (TypeError, "k or v is", (q, k.float(), v.float(), cu)),
            (TypeError, "int32", (q, k, v, cu.long())),
            (ValueError, "1-dimensional", (q, k, v, cu[None])),
            (ValueError, "one entry more", (q, k, v, cu[:0])),
            (ValueError, "scale must be positive", (q, k, v, cu, 0.0)),
            (ValueError, "scale must be positive", (q, k, v, cu, math.nan)),
            (ValueError, "scale must be positive", (q, k, v, cu, 1e-50)),
            (ValueError, "scale must be positive", (q, k, v, cu, 1e50)),
            (ValueError, "65536 sequences", (q, k, v, cu.new_zeros(65538)))]:
        with pytest.raises(err, match=match):
            f(*args)


@pytest.mark.parametrize("dev", DEVS)
def test_huge_scores(dev):
    """Scores near the end of the range on either side, all of one sign: the
    mean of the values, not zeros."""
    q, k, v, _ = _inputs([70, 300], 0, 4, 2, 64, dev)
    for sign in (-1, 1):
        o = ops.flash_attention_packed(
            torch.full_like(q, 2.0 ** 60), torch.full_like(k, sign * 2.0 ** 60),
            torch.full_like(v, 1.5), _cu([70, 300], dev))
        assert torch.equal(o, torch.full_like(o, 1.5))


@pytest.mark.parametrize("dev", DEVS)
def test_as_many_sequences_as_are_taken(dev):
    """65536 sequences, all but a few of them empty."""
    lens = [0] * 65536
    for b, n in ((0, 3), (63, 1), (64, 40), (40000, 7), (65535, 300)):
        lens[b] = n
    q, k, v, go = _inputs([351], 5, 4, 2, 64, dev)
    qkv = [t.requires_grad_(True) for t in (q, k, v)]
    o = ops.flash_attention_packed(*qkv, _cu(lens, dev))
    got = (o, *torch.autograd.grad(o, qkv, go))
    _check(got, *_oracle(q, k, v, go, [n for n in lens if n], 64 ** -0.5))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("D", [64, 192])
def test_more_sequences_than_lanes(dev, D):
    """Many sequences of one block, a few of many, empty ones between them."""
    lens = [(7 * b) % 23 for b in range(75)]
    lens[3], lens[70], lens[74] = 1300, 129, 257
    q, k, v, go = _inputs(lens, 9, 2, 1, D, dev)
    _check(_run(q, k, v, go, _cu(lens, dev)),
           *_oracle(q, k, v, go, lens, D ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[131200, 1, 60, 0, 300], [5, 700, 0, 2000]])
def test_listed_blocks_give_the_same_bits(lens):
    """The same sequences with empty ones behind them, past 64, and past the
    levels that the list tells apart."""
    q, k, v, go = _inputs(lens, 3, 2, 1, 64, "cuda")
    a = _run(q, k, v, go, _cu(lens, "cuda"))
    b = _run(q, k, v, go, _cu(lens + [0] * 70, "cuda"))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 53])
def test_gradient_is_taken_once(D):
    q, k, v, go = _inputs([20, 30], 0, 4, 2, D, "cuda")
    cu = _cu([20, 30], "cuda")
    q = q.requires_grad_(True)               # k and v need none
    o = ops.flash_attention_packed(q, k, v, cu)
    plain, = torch.autograd.grad(o, q, go, retain_graph=True)
    dq, = torch.autograd.grad(o, q, go, create_graph=True)
    assert torch.equal(plain, dq) and dq.requires_grad
    # (the copies of rows of 53 do not lead back to q)
    with pytest.raises(RuntimeError,
                       match="once" if D == 64 else "not have been used"):
        torch.autograd.grad(dq.sum(), q)
    assert torch.equal(plain, _run(q, k, v, go, cu)[1])
    # checkpointing runs the forward again
    c = torch.utils.checkpoint.checkpoint(
        lambda *a: ops.flash_attention_packed(*a), q, k, v, cu,
        use_reentrant=False)
    again, = torch.autograd.grad(c, q, go)
    assert torch.equal(plain, again)


def test_border_refusals_on_the_cpu():
    q, k, v, _ = _inputs([6], 0, 4, 2, 64, "cpu")
    for cu in ([0, 7], [1, 6], [0, 4, 2]):
        with pytest.raises(ValueError, match="must rise"):
            ops.flash_attention_packed(q, k, v,
                                       torch.tensor(cu, dtype=torch.int32))


@pytest.mark.gpu
def test_gpu_refusals():
    q, k, v, _ = _inputs([6], 0, 4, 2, 64, "cuda")
    cu = _cu([6], "cuda")
    with pytest.raises(TypeError, match="bf16"):
        ops.flash_attention_packed(q.float(), k.float(), v.float(), cu)
    with pytest.raises(ValueError, match="cu_seqlens is on cpu"):
        ops.flash_attention_packed(q, k, v, cu.cpu())


@pytest.mark.gpu
def test_matches_the_dense_kernel():
    """Sequences of one length are the dense op's batch."""
    B, S, H, HKV, D = 3, 200, 6, 2, 159
    q, k, v, go = _inputs([S] * B, 0, H, HKV, D, "cuda")
    o = ops.flash_attention_packed(q, k, v, _cu([S] * B, "cuda"))
    dense = ops.flash_attention(q.reshape(B, S, H, D), k.reshape(B, S, HKV, D),
                                v.reshape(B, S, HKV, D))
    val, tol = _oracle(q, k, v, go, [S] * B, D ** -0.5)
    # the dense kernel rounds the scaled q to bf16 as well
    assert ((dense.reshape(B * S, H, D).double().cpu() - val[0]).abs()
            <= 8 * tol[0]).all()
    _check((o,), val, tol)


@pytest.mark.gpu
def test_capture_and_replay():
    """Forward and backward captured; borders and inputs change between the
    replays, with eager calls on other leaves beside them."""
    T, H, HKV, D = 400, 4, 2, 96
    q, k, v, go = _inputs([T], 0, H, HKV, D, "cuda")
    cu = _cu([100, 250, 50], "cuda")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]

    def step(x):
        o = ops.flash_attention_packed(*x, cu)
        return (o.detach(), *torch.autograd.grad(o, x, go))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(leaves)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaves)
    for i, lens in enumerate(([400, 0, 0], [1, 2, 390], [133, 133, 134])):
        cu.copy_(_cu(lens, "cpu"))
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn_like(t))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        eager = step([t.detach().clone().requires_grad_(True)
                      for t in leaves])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


@pytest.mark.gpu
def test_borders_out_of_range_stay_inside():
    """Contents that the host cannot see lead nowhere outside the tensors: the
    rows before and behind the buffers keep their values."""
    T, H, HKV, D = 64, 2, 1, 64
    room = torch.full((3 * T, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    q, k, v, go = _inputs([T], 0, H, HKV, D, "cuda")
    room[T:2 * T] = q
    for cu in ([0, 10 ** 9], [-50, 64], [5, 20, 64], [0, 40, 20, 64],
               [0, -1, 64], [0, 64] * 50, [5] * 90 + [100], [64, 0] * 50,
               [-9, 2 ** 31 - 1] * 50, list(range(200, 0, -1))):
        c = torch.tensor(cu, dtype=torch.int32, device="cuda")
        _run(room[T:2 * T], k, v, go, c)
    torch.cuda.synchronize()
    assert (room[:T] == 7).all() and (room[2 * T:] == 7).all()


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls under way on two streams, over the list of blocks and without it."""
    sides = []
    for seed, lens in ((0, [700, 3, 520]), (1, [9] * 90)):
        q, k, v, go = _inputs(lens, 4, 4, 2, 96, "cuda", seed=seed)
        cu = _cu(lens, "cuda")
        sides.append((q, k, v, go, cu, _run(q, k, v, go, cu)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    got = [[], []]
    for _ in range(8):
        for out, st, (q, k, v, go, cu, _ref) in zip(got, streams, sides):
            with torch.cuda.stream(st):
                out.append(_run(q, k, v, go, cu))
    torch.cuda.synchronize()
    for outs, side in zip(got, sides):
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, side[-1]))
