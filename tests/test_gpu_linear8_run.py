"""The operators as they are used together: a mixture-of-experts block in 8 bits from the residual stream to the combined output, one token and
batches, against the same chain in 64 bits from the codes that the chain itself produced; and a training step of the routing around bf16 experts."""
import pytest
import torch

import kernelschema_b200 as ks

pytestmark = pytest.mark.gpu

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def weights8(e, n, k, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(e, n, k, generator=g, device="cuda") * 0.05
    s = w.abs().amax(dim=-1) / TOP[dtype]
    q = w / s[..., None]
    return (q.round() if dtype == torch.int8 else q).to(dtype), s


def block(x, r, gain, gate, w1, s1, w2, s2, top_k, dtype):
    """One pre-norm expert block; returns every intermediate."""
    q, qs, hidden, normed = ks.rmsnorm_quantize(x, gain, r, 1e-6, dtype, normed=True)
    ids, w = ks.route_topk(ks.router_logits(normed, gate), top_k)
    order = ks.route_sort(ids, gate.shape[0])
    rows, rs = ks.sort_tokens(q, order), ks.sort_tokens(qs, order)
    up = ks.mm_8bit_grouped(rows, rs, w1, s1, order.offsets)
    a, as_ = ks.swiglu_quantize(up, dtype)
    down = ks.mm_8bit_grouped(a, as_, w2, s2, order.offsets)
    return dict(q=q, qs=qs, hidden=hidden, normed=normed, ids=ids, w=w, order=order, rows=rows, rs=rs, up=up, a=a, as_=as_, down=down,
                y=ks.unsort_tokens(down, order, w))


@pytest.mark.parametrize("dtype", TOP)
@pytest.mark.parametrize("t", (1, 5, 64, 700))
def test_expert_block(t, dtype):
    h, i, e, top_k = 512, 200, 16, 4
    i16 = i // 16 * 16
    g = torch.Generator(device="cuda").manual_seed(t)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, r, gain, gate = rand(t, h).bfloat16(), rand(t, h).bfloat16(), (1 + 0.1 * rand(h)).bfloat16(), (rand(e, h) * 0.05).bfloat16()
    (w1, s1), (w2, s2) = weights8(e, 2 * i16, h, dtype, 1), weights8(e, h, i16, dtype, 2)
    got = block(x, r, gain, gate, w1, s1, w2, s2, top_k, dtype)
    assert torch.equal(got["hidden"], (x.float() + r.float()).bfloat16())
    # the experts, token by token, from the chain's own codes and selection
    ids, w = got["ids"].long(), got["w"].double()
    xin = got["q"].double() * got["qs"].double()[:, None]
    y = torch.zeros(t, h, dtype=torch.float64, device="cuda")
    size = torch.zeros(t, h, dtype=torch.float64, device="cuda")
    for k in range(top_k):
        m1, m2 = w1[ids[:, k]].double() * s1[ids[:, k]].double()[..., None], w2[ids[:, k]].double() * s2[ids[:, k]].double()[..., None]
        up = torch.einsum("th,tnh->tn", xin, m1)
        act = up[:, :i16] * torch.sigmoid(up[:, :i16]) * up[:, i16:]
        y += torch.einsum("tn,thn->th", act, m2) * w[:, k:k + 1]
        # what roundings move: `up` to bf16 (2^-8 of it: 3 * 2^-8 of the product of its halves, the gate's slope being at most 1.1 per unit), a code by half a
        # step (of amax / 127, or 2^-4 of its size and half of the least step, which 2^-10 of amax / 448 bounds), `down` and y to bf16
        step = act.abs().amax(dim=1, keepdim=True) * (0.5 / 127 if dtype == torch.int8 else 2.0 ** -10 / 448) + (0.0 if dtype == torch.int8 else 2.0 ** -4) * act.abs()
        moved = step + (up[:, :i16].abs() * up[:, i16:].abs() * 1.1 + act.abs()) * 2.0 ** -8 * 1.01
        size += (torch.einsum("tn,thn->th", moved, m2.abs()) + 2.0 ** -8 * torch.einsum("tn,thn->th", act.abs(), m2.abs())) * w[:, k:k + 1]
    off = (got["y"].double() - y).abs()
    assert bool((off <= size * 1.05 + y.abs() * 2.0 ** -8 + 1e-6).all()), float((off - size).max())
    # dense products of the same rows, and the chain captured and replayed on other tokens
    assert torch.equal(ks.mm_8bit(got["q"], got["qs"], w1[3], s1[3]), ks.mm_8bit_grouped(got["q"], got["qs"], w1[3:4], s1[3:4], torch.tensor([0, t], dtype=torch.int32, device="cuda"))) \
        or dtype != torch.int8
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = block(x, r, gain, gate, w1, s1, w2, s2, top_k, dtype)
    x.copy_(rand(t, h).bfloat16())
    graph.replay()
    want = block(x, r, gain, gate, w1, s1, w2, s2, top_k, dtype)
    for name in ("q", "qs", "hidden", "normed", "ids", "w", "rows", "rs", "up", "a", "as_", "down", "y"):
        assert torch.equal(again[name].view(torch.uint8) if again[name].dtype == torch.float8_e4m3fn else again[name],
                           want[name].view(torch.uint8) if want[name].dtype == torch.float8_e4m3fn else want[name]), name


def test_training_step_around_experts():
    """Gradients of a routed layer with bf16 experts between sort and unsort, against the same step in fp64 per token."""
    t, h, e, top_k = 96, 64, 8, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w = rand(t, h).requires_grad_(), rand(t, top_k).softmax(dim=1).requires_grad_()
    experts, dy = (rand(e, h, h) * 0.1).requires_grad_(), rand(t, h)
    ids = torch.rand(t, e, generator=g, device="cuda").topk(top_k, dim=1).indices.int()
    ids[5] = -1                                              # a token whose experts are elsewhere
    order = ks.route_sort(ids, e)
    rows = ks.sort_tokens(x, order)
    at = order.offsets.tolist()
    products = torch.cat([rows[at[i]:at[i + 1]] @ experts[i] for i in range(e)] + [rows[at[e]:]])
    grads = torch.autograd.grad(ks.unsort_tokens(products, order, w), (x, w, experts), dy)
    xd, wd, ed = (v.detach().double().requires_grad_() for v in (x, w, experts))
    there = (ids >= 0)
    y = sum(torch.where(there[:, k:k + 1], torch.einsum("th,thn->tn", xd, ed[ids[:, k].clamp(min=0).long()]) * wd[:, k:k + 1], 0.0) for k in range(top_k))
    for got, want in zip(grads, torch.autograd.grad(y, (xd, wd, ed), dy.double())):
        # fp32 sums of at most a few hundred terms, in two products and the operators' own; torch's matmul may use TF32 nowhere (default)
        assert float((got.double() - want).abs().max()) <= 1e-4 * float(want.abs().max())
    assert not bool(grads[0][5].any()) and not bool(grads[1][5].any())
