"""Golden tests for the gather-only MoE dispatch/combine path against a
naive differentiable reference (the semantics the first implementation and
the reference model.py:1219-1242 define)."""

import pytest
import torch

from luminaai_amd.ops.interface import (moe_combine, moe_dispatch,
                                        moe_routing_plan)


def _naive(xf, topi, topw, E, C):
    """index_put/index_add formulation (slow, pure autograd)."""
    N, k = topi.shape
    h = xf.shape[1]
    flat_e = topi.reshape(-1)
    order = torch.argsort(flat_e, stable=True)
    tok = torch.div(order, k, rounding_mode="floor")
    counts = torch.bincount(flat_e, minlength=E)
    offs = torch.cumsum(counts, 0) - counts
    sorted_e = flat_e[order]
    pos = torch.arange(N * k) - offs[sorted_e]
    valid = pos < C
    dest = torch.where(valid, sorted_e * C + pos, torch.full_like(pos, E * C))
    buf = xf.new_zeros(E * C + 1, h)
    buf = torch.index_put(buf, (dest,), xf[tok])
    bufv = buf[:E * C]
    # identity "expert computation" so combine is testable end to end
    y = bufv * 2.0 + 1.0
    gathered = y.reshape(E * C, h)[dest.clamp_max(E * C - 1)]
    w_sorted = (topw.reshape(-1)[order] * valid.float())
    out = xf.new_zeros(N, h).index_add(0, tok, gathered * w_sorted.unsqueeze(1))
    return bufv, out


@pytest.mark.parametrize("seed,cap_frac", [(0, 1.25), (1, 0.5), (2, 10.0)])
def test_dispatch_combine_matches_naive(seed, cap_frac):
    torch.manual_seed(seed)
    N, h, E, k = 64, 16, 4, 2
    C = max(1, int(N * k / E * cap_frac))
    xf = torch.randn(N, h, requires_grad=True)
    xf2 = xf.detach().clone().requires_grad_(True)
    logits = torch.randn(N, E)
    topw, topi = logits.softmax(-1).topk(k, dim=-1)
    topw = (topw / topw.sum(-1, keepdim=True)).detach()
    w1 = topw.clone().requires_grad_(True)
    w2 = topw.clone().requires_grad_(True)

    buf_ref, out_ref = _naive(xf, topi, w1, E, C)

    plan = moe_routing_plan(topi, E, C)
    buf = moe_dispatch(xf2, plan).view(E, C, h)
    torch.testing.assert_close(buf, buf_ref.view(E, C, h))
    y = (buf.reshape(E * C, h) * 2.0 + 1.0)
    out = moe_combine(y, w2.reshape(-1), plan)
    torch.testing.assert_close(out, out_ref)

    g = torch.randn_like(out)
    out_ref.backward(g)
    out.backward(g)
    torch.testing.assert_close(xf2.grad, xf.grad, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(w2.grad, w1.grad, rtol=1e-5, atol=1e-6)


def test_dropped_tokens_get_zero_weight():
    torch.manual_seed(0)
    N, h, E, k = 8, 4, 2, 1
    C = 2  # only 2 slots per expert -> drops guaranteed
    topi = torch.zeros(N, 1, dtype=torch.long)  # everyone wants expert 0
    topw = torch.ones(N, 1)
    plan = moe_routing_plan(topi, E, C)
    assert int(plan.fill_mask.sum()) == 2      # capacity respected
    xf = torch.randn(N, h)
    buf = moe_dispatch(xf, plan)
    torch.testing.assert_close(buf[:2], xf[:2])       # stable order: first wins
    assert buf[2:].abs().sum() == 0
    out = moe_combine(buf, topw.reshape(-1), plan)
    torch.testing.assert_close(out[:2], xf[:2])
    assert out[2:].abs().sum() == 0                    # dropped -> zero output


def test_plan_counts():
    topi = torch.tensor([[0], [0], [1], [3]])
    plan = moe_routing_plan(topi, 4, 8)
    assert plan.counts.tolist() == [2, 1, 0, 1]


@pytest.mark.parametrize("dev", ["cpu", pytest.param(
    "cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("k", [1, 2, 3])
def test_limits_of_each_sequence(dev, k):
    """Each sequence keeps what a plan of it alone keeps."""
    torch.manual_seed(k)
    E, lens = 4, [1, 9, 0, 30, 2, 17]
    N = sum(lens)
    topi = torch.stack([torch.randperm(E)[:k] for _ in range(N)])
    topi[:20, 0] = 1
    limit = torch.tensor([max(1, -(-n * k * 5 // (E * 4))) for n in lens])
    seq = torch.repeat_interleave(torch.arange(6), torch.tensor(lens))
    C = int(limit.sum())
    plan = moe_routing_plan(topi.to(dev), E, C, seq.to(dev), limit.to(dev))
    slot = plan.slot_tm.cpu().view(N, k)
    at = 0
    for n, most in zip(lens, limit.tolist()):
        if n:
            alone = moe_routing_plan(topi[at:at + n], E, most)
            kept = alone.slot_tm.view(n, k) < E * most
            assert torch.equal(slot[at:at + n] < E * C, kept)
        at += n
    kept = slot < E * C
    assert torch.equal(slot[kept] // C, topi[kept])     # in the right bucket
    assert slot[kept].unique().numel() == int(kept.sum())
    fill = plan.fill_mask.cpu().nonzero()[:, 0]
    assert torch.equal(fill, slot[kept].sort().values)
    assert torch.equal(plan.inv.cpu()[slot[kept]],
                       torch.arange(N * k).view(N, k)[kept])
    assert torch.equal(plan.counts.cpu(),
                       torch.bincount(topi.reshape(-1), minlength=E))


@pytest.mark.parametrize("C", [1, 5, 40])
def test_limits_with_any_sequence_numbers(C):
    """Numbers that fall, and limits past the bucket, lead nowhere outside."""
    torch.manual_seed(0)
    topi = torch.randint(0, 4, (50, 2))
    seq = torch.randint(0, 7, (50,))
    plan = moe_routing_plan(topi, 4, C, seq, torch.full((7,), 9))
    assert 0 <= int(plan.slot_tm.min()) and int(plan.slot_tm.max()) <= 4 * C
    kept = plan.slot_tm[plan.slot_tm < 4 * C]
    assert kept.unique().numel() == kept.numel() == int(plan.fill_mask.sum())
