"""token_logprobs against 64-bit forms, on the CPU path and on the kernels."""

import math

import pytest
import torch

from luminaai_amd import ops

DEVS = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
EPS = 2.0 ** -24


def _oracle(x, tok, k, ignore=-100):
    x = x.detach().double().cpu()
    tok = tok.cpu().long()
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
    rows = torch.arange(x.shape[0])
    inside = (tok >= 0) & (tok < x.shape[1])
    lp = logp[rows, tok.clamp(0, x.shape[1] - 1)]
    lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
    lp = torch.where(tok == ignore, torch.zeros_like(lp), lp)
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
    return lp, ent, torch.take_along_dim(logp, ids, 1), ids


def _tol(V, lp):
    """fp32: a thread adds V / 512 + 40 terms, each off by its exponent's
    rounding (a term 2^-y has y EPS relative, at most 1.1 in sum for y 2^-y)
    and one step; the logarithm and the last two differences a step each of
    what they hold (under 128)."""
    return EPS * (V / 512 + 48) + 4 * EPS * (lp.abs() + 32)


def _check(r, x, tok, k):
    lp, ent, tl, ids = _oracle(x, tok, k)
    V = x.shape[1]
    got = [t.detach().double().cpu() for t in r[:3]]
    fine = lp.isfinite()
    assert torch.equal(got[0].isnan(), lp.isnan())
    assert ((got[0] - lp).abs()[fine] <= _tol(V, lp)[fine]).all()
    assert torch.equal(got[0][~fine & ~lp.isnan()], lp[~fine & ~lp.isnan()])
    # the entropy is a mean of at most log V + 1 of such values
    assert ((got[1] - ent).abs() <= (2 + math.log(V)) * _tol(V, ent)).all()
    assert torch.equal(r.top_ids.cpu(), ids)
    fin = tl.isfinite()
    assert ((got[2] - tl).abs()[fin] <= _tol(V, tl)[fin]).all()
    assert torch.equal(got[2][~fin], tl[~fin])


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
@pytest.mark.parametrize("V,k", [(1, 1), (7, 7), (63, 5), (100, 64),
                                 (1024, 20), (4099, 32), (50304, 20),
                                 (50257, 0)])
def test_token_logprobs(dev, dtype, V, k):
    g = torch.Generator().manual_seed(V)
    x = (2.5 * torch.randn(9, V, generator=g)).to(dtype).to(dev)
    tok = torch.randint(0, V, (9,), generator=g).to(dev)
    tok[3] = -100
    _check(ops.token_logprobs(x, tok, k), x, tok, k)
    _check(ops.token_logprobs(x, tok.int(), k), x, tok, k)


@pytest.mark.parametrize("dev", DEVS)
def test_shapes_and_strides(dev):
    x = torch.randn(3, 5, 2, 70, device=dev)
    tok = torch.randint(0, 70, (3, 5, 2), device=dev)
    r = ops.token_logprobs(x, tok, 3)
    assert r.logprobs.shape == (3, 5, 2) and r.top_ids.shape == (3, 5, 2, 3)
    flat = ops.token_logprobs(x.reshape(-1, 70), tok.reshape(-1), 3)
    assert torch.equal(r.top_ids.view(-1, 3), flat.top_ids)
    # the last position of each row of a batch, channels apart
    last = ops.token_logprobs(x[:, -1, 0], tok[:, -1, 0], 3)
    assert torch.equal(last.logprobs, r.logprobs[:, -1, 0])
    xt = x[:, :, 0, :].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(ops.token_logprobs(xt, tok[..., 0]).entropy,
                       r.entropy[..., 0])
    one = ops.token_logprobs(x[0, 0, 0], tok[0, 0, 0], 3)
    assert one.logprobs.shape == () and one.top_ids.shape == (3,)
    assert torch.equal(one.logprobs, r.logprobs[0, 0, 0])
    none = ops.token_logprobs(x[:0], tok[:0], 3)
    assert none.top_ids.shape == (0, 5, 2, 3)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
def test_masks(dev, dtype):
    """Logits of -inf and of the type's lowest value, in part and throughout."""
    V = 3001
    low = torch.finfo(dtype).min
    x = torch.randn(6, V).to(dtype)
    x[0, 100:] = -math.inf
    x[1, 100:] = low
    x[2, :] = low                                  # uniform
    x[3, :] = -math.inf
    x[3, 77] = 2.0                                 # certain
    x[4, 1::2] = -math.inf
    x = x.to(dev)
    tok = torch.tensor([5, 5, 9, 77, 1, 0], device=dev)
    _check(ops.token_logprobs(x, tok, 64), x, tok, 64)
    r = ops.token_logprobs(x, tok)
    assert float(r.logprobs[4]) == -math.inf and float(r.entropy[3]) == 0


@pytest.mark.parametrize("dev", DEVS)
def test_rows_without_distribution(dev):
    x = torch.randn(4, 900, device=dev)
    x[0] = -math.inf
    x[1, 5] = math.nan
    x[2, 7] = math.inf
    tok = torch.tensor([1, 2, 3, 4], device=dev)
    r = ops.token_logprobs(x, tok, 4)
    assert r.logprobs.isnan().tolist() == [True, True, True, False]
    assert r.entropy.isnan().tolist() == [True, True, True, False]
    assert r.top_ids[0].tolist() == [0, 1, 2, 3]
    assert int(r.top_ids[1, 0]) == 5 and int(r.top_ids[2, 0]) == 7
    rest = x[1].clone()
    rest[5] = -math.inf
    assert torch.equal(r.top_ids[1, 1:], rest.topk(3).indices)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties_take_the_lowest_index(dev, dtype):
    V = 6007
    x = torch.zeros(5, V, dtype=dtype)
    x[1] = torch.randint(0, 3, (V,)).to(dtype)          # thousands of ties
    x[2, 4000] = 1.0
    x[3, ::2] = -0.0                                    # equal to 0
    x[4] = torch.arange(V).div(50, rounding_mode="floor").neg().to(dtype)
    x = x.to(dev)
    tok = torch.zeros(5, dtype=torch.long, device=dev)
    _check(ops.token_logprobs(x, tok, 64), x, tok, 64)


@pytest.mark.parametrize("dev", DEVS)
def test_tokens_outside(dev):
    x = torch.randn(5, 40, device=dev, requires_grad=True)
    tok = torch.tensor([-100, -1, 40, 2 ** 40, 3], device=dev)
    r = ops.token_logprobs(x, tok)
    assert r.logprobs.isnan().tolist() == [False, True, True, True, False]
    assert float(r.logprobs[0]) == 0
    assert r.entropy.isfinite().all()
    dx, = torch.autograd.grad(r.logprobs[[0, 4]].sum(), x)
    assert (dx[0] == 0).all() and dx[4].abs().sum() > 0
    keep = ops.token_logprobs(x, torch.tensor([7, 7, 7, 7, 3], device=dev),
                              ignore_index=7)
    assert keep.logprobs[:4].eq(0).all() and float(keep.logprobs[4]) != 0


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16,
                                   torch.float32])
@pytest.mark.parametrize("V", [5, 1024, 9001, 50304])
@pytest.mark.parametrize("which", ["both", "lp", "ent"])
def test_gradient(dev, dtype, V, which):
    """Against autograd through the formula in 64 bits."""
    g = torch.Generator().manual_seed(V)
    N = 4
    x = (2.5 * torch.randn(N, V, generator=g)).to(dtype)
    x[1, V // 2:] = -math.inf
    tok = torch.randint(0, max(1, V // 2), (N,), generator=g)
    tok[2] = -100
    gl, ge = torch.randn(2, N, generator=g)
    if which == "lp":
        ge = ge * 0
    elif which == "ent":
        gl = gl * 0
    xr = x.double().requires_grad_(True)
    logp = torch.log_softmax(xr, -1)
    ent = -(logp.exp() * logp.masked_fill(logp == -math.inf, 0)).sum(-1)
    lp = logp[torch.arange(N), tok.clamp(min=0)] * (tok != -100)
    want, = torch.autograd.grad((lp * gl).sum() + (ent * ge).sum(), xr)

    xd = x.to(dev).requires_grad_(True)
    r = ops.token_logprobs(xd, tok.to(dev), 3)
    assert not r.top_logprobs.requires_grad
    outs, gs = {"both": ([r.logprobs, r.entropy], [gl, ge]),
                "lp": ([r.logprobs], [gl]),
                "ent": ([r.entropy], [ge])}[which]
    dx, = torch.autograd.grad(outs, xd, [t.to(dev) for t in gs])
    assert dx.dtype == dtype
    # the one rounding to the type (fp16 also below its smallest normal
    # number), and fp32 values off by what p, H and y are off (_tol, times
    # p (|gl| + |ge| (|log p| + H + 1)))
    p = logp.detach().exp()
    y = logp.detach().masked_fill(p == 0, 0).abs()
    size = gl.abs()[:, None] + ge.abs()[:, None] * (y + ent.detach()[:, None]
                                                    + 1)
    tol = want.abs() * (torch.finfo(dtype).eps / 2) + 4 * p * size * (
        _tol(V, y) * (2 + math.log(V)))
    tol += torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    tol[torch.arange(N), tok.clamp(min=0)] += gl.abs().double() * 2 * EPS
    assert ((dx.double().cpu() - want).abs() <= tol).all()
    assert (dx[1, V // 2:] == 0).all()


@pytest.mark.parametrize("dev", DEVS)
def test_gradient_against_differences(dev):
    """f(x + h d) - f(x - h d) over 2 h, f summed in 64 bits. With |d| <= 1 the
    third derivative of log softmax and entropy along d is under 40 a row, so
    the difference is off by 40 N h^2 / 6, and by f's rounding (_tol) / h."""
    g = torch.Generator().manual_seed(2)
    N, V, h = 6, 300, 2.0 ** -6
    x = (2 * torch.randn(N, V, generator=g)).to(dev)
    d = (2 * torch.rand(N, V, generator=g) - 1).to(dev)
    tok = torch.randint(0, V, (N,), generator=g).to(dev)

    def f(z):
        r = ops.token_logprobs(z, tok)
        return (r.logprobs.double().sum() + r.entropy.double().sum())

    xg = x.clone().requires_grad_(True)
    r = ops.token_logprobs(xg, tok)
    dx, = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), xg)
    slope = float((dx.double() * d.double()).sum())
    diff = float(f(x + h * d) - f(x - h * d)) / (2 * h)
    bound = 40 * N * h * h / 6 + N * (3 + math.log(V)) * float(
        _tol(V, torch.tensor(12.0))) / h + N * V * EPS * 16
    assert abs(slope - diff) <= bound


@pytest.mark.parametrize("dev", DEVS)
def test_refusals(dev):
    x = torch.randn(4, 30, device=dev)
    tok = torch.zeros(4, dtype=torch.long, device=dev)
    with pytest.raises(ValueError, match="do not match"):
        ops.token_logprobs(x, tok[:3])
    with pytest.raises(ValueError, match="top_k"):
        ops.token_logprobs(x, tok, 31)
    with pytest.raises(ValueError, match="top_k"):
        ops.token_logprobs(x.repeat(1, 9), tok, 65)
    with pytest.raises(ValueError, match="top_k"):
        ops.token_logprobs(x, tok, -1)
    with pytest.raises(TypeError, match="int64 or int32"):
        ops.token_logprobs(x, tok.float())
    with pytest.raises(TypeError, match="bf16, fp16 or fp32"):
        ops.token_logprobs(x.int(), tok)
    with pytest.raises(ValueError, match="rows, vocab"):
        ops.token_logprobs(x[:, :0], tok)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-math.inf, "lowest", -1e30, 0.0, -0.0])
def test_alternatives_among_many_equal(dev, dtype, mask):
    """Rows with few tokens beside a mask: the first masked tokens follow."""
    V, N, k = 9003, 6, 20
    g = torch.Generator().manual_seed(0)
    mask = torch.finfo(dtype).min if mask == "lowest" else mask
    x = torch.full((N, V), mask).to(dtype)
    some = torch.randn(N, 5, generator=g).to(dtype)
    x[0, 100:105] = some[0]
    x[1, [0, 7, 8999, 9000, 9002]] = some[1]
    x[2, 8000:] = torch.randn(1003, generator=g).to(dtype)
    x[3, :8990] = -math.inf                   # the mask's equals come last
    x[4, ::64] = 1.0                          # more equals than fit, above it
    x[5, torch.arange(V) // 8 % 64 != 5] = torch.randn(
        int((torch.arange(V) // 8 % 64 != 5).sum()), generator=g).to(dtype)
    for kk in (1, k, 64):
        r = ops.token_logprobs(x.to(dev), torch.zeros(N, dtype=torch.long,
                                                      device=dev), kk)
        # falling value, then index (the two zeros are equal)
        order = torch.sort(x.double() + 0.0, dim=1, descending=True,
                           stable=True).indices[:, :kk]
        assert torch.equal(r.top_ids.cpu(), order)


def _nan_first(x, k):
    """Alternatives with NaN above all, then falling values, ties to the lowest
    index."""
    x = x.double() + 0.0
    key = torch.where(x.isnan(), math.inf, x)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    last = torch.sort(x.isnan().gather(1, order).int(), dim=1, descending=True,
                      stable=True).indices
    return order.gather(1, last)[:, :k]


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alternatives_of_many_nan(dev, dtype):
    """More NaN than fit beside each other, from the first token on."""
    V = 3000
    x = torch.randn(4, V, generator=torch.Generator().manual_seed(0))
    x[0] = math.nan
    x[1, :1500] = math.nan
    x[2, 1:1500] = math.nan
    x[3, ::2] = math.nan
    x = x.to(dtype)
    tok = torch.zeros(4, dtype=torch.long, device=dev)
    for k in (1, 3, 64):
        r = ops.token_logprobs(x.to(dev), tok, k)
        assert torch.equal(r.top_ids.cpu(), _nan_first(x, k))
        assert r.top_logprobs.isnan().all()


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-math.inf, -1e30, 0.0])
def test_alternatives_beside_a_nan_and_a_mask(dev, dtype, mask):
    """A NaN early in the row, larger logits beside it and elsewhere, and more
    equal logits than fit."""
    V, k = 50304, 20
    x = torch.full((4, V), mask).to(dtype)
    x[0, 3] = math.nan
    x[0, 5], x[0, 20], x[0, 50303] = 2.0, 1.0, 3.0
    x[1, 40000] = math.nan
    x[1, 40001] = 1.5
    x[2, [0, 9000, 50303]] = math.nan
    x[2, 30] = math.inf
    x[3, ::4096] = math.nan
    x[3, 1::4096] = 1.0
    tok = torch.zeros(4, dtype=torch.long, device=dev)
    for kk in (1, k, 64):
        r = ops.token_logprobs(x.to(dev), tok, kk)
        assert torch.equal(r.top_ids.cpu(), _nan_first(x, kk))


@pytest.mark.gpu
def test_gradient_is_taken_once():
    x = torch.randn(5, 700, device="cuda", requires_grad=True)
    tok = torch.randint(0, 700, (5,), device="cuda")
    r = ops.token_logprobs(x, tok)
    plain, = torch.autograd.grad(r.logprobs.sum(), x, retain_graph=True)
    dx, = torch.autograd.grad(r.logprobs.sum(), x, create_graph=True)
    assert torch.equal(plain, dx) and dx.requires_grad
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(dx.sum(), x)
    # only the alternatives are used: no gradient reaches the logits
    assert not ops.token_logprobs(x, tok, 3).top_logprobs.requires_grad


@pytest.mark.gpu
def test_capture_and_replay():
    x = torch.randn(40, 5000, device="cuda").bfloat16().requires_grad_(True)
    tok = torch.randint(0, 5000, (40,), device="cuda")
    gl = torch.randn(40, device="cuda")

    def step():
        r = ops.token_logprobs(x, tok, 5)
        dx, = torch.autograd.grad([r.logprobs, r.entropy], x, [gl, gl])
        return r.logprobs.detach(), r.entropy.detach(), r.top_ids, dx

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(40, 5000, device="cuda") * (i + 1))
            tok.copy_(torch.randint(0, 5000, (40,), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """More than 2^32 logits: the last rows."""
    V, N = 131072, 33000
    x = torch.empty(N, V, dtype=torch.bfloat16, device="cuda")
    x.zero_()
    x[-2:] = torch.randn(2, V, device="cuda").bfloat16()
    tok = torch.full((N,), 9, device="cuda")
    r = ops.token_logprobs(x, tok, 2)
    want = ops.token_logprobs(x[-2:].clone(), tok[-2:], 2)
    for a, b in zip(r, want):
        assert torch.equal(a[-2:], b)


@pytest.mark.gpu
def test_gpu_refuses_rows_past_its_indexes():
    x = torch.empty(1, 2 ** 30 + 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="not supported"):
        ops.token_logprobs(x, torch.zeros(1, dtype=torch.long, device="cuda"))
