"""Tokens sorted by expert and back, and their gradients, against definitions in plain Python and 64 bits."""
import pytest
import torch

import kernelschema_b200 as ks

pytestmark = pytest.mark.gpu

KINDS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make_ids(t, k, e, seed, masked=0.2, distinct=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if distinct:
        return torch.rand(t, e, generator=g, device="cuda").topk(k, dim=1).indices.int()
    ids = torch.randint(0, e, (t, k), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand(t, k, generator=g, device="cuda")
    return torch.where(u < masked / 2, -1, torch.where(u < masked, ids + e, ids)).int()


def expected_order(ids, e):
    flat = ids.flatten().tolist()
    by = sorted((i for i, v in enumerate(flat) if 0 <= v < e), key=lambda i: flat[i])
    offsets, row_of = [0] * (e + 1), [-1] * len(flat)
    for row, i in enumerate(by):
        row_of[i] = row
        offsets[flat[i] + 1] += 1
    for i in range(e):
        offsets[i + 1] += offsets[i]
    return offsets, row_of, by + [-1] * (len(flat) - len(by))


def check_order(ids, e):
    order = ks.route_sort(ids, e)
    offsets, row_of, route_of_row = expected_order(ids, e)
    assert order.offsets.tolist() == offsets
    assert order.row_of.flatten().tolist() == row_of and order.row_of.shape == ids.shape
    assert order.route_of_row.tolist() == route_of_row
    return order


# one block, the one-launch form up to 8192 routes, the two- and (above 131072 routes) the three-launch form; experts around powers of two
@pytest.mark.parametrize("t,k,e", [(0, 8, 4), (1, 1, 1), (1, 8, 256), (3, 2, 1), (32, 8, 128), (33, 31, 7), (127, 8, 1023), (128, 8, 1024), (129, 8, 64), (1024, 8, 128),
                                   (1025, 8, 127), (1777, 8, 128), (5000, 3, 65), (8192, 8, 256), (16384, 8, 31), (16385, 8, 33), (20011, 11, 1024)])
def test_order(t, k, e):
    check_order(make_ids(t, k, e, t + k + e), e)


def test_order_edges():
    for t, k in ((5, 3), (3000, 4)):
        check_order(torch.full((t, k), -1, dtype=torch.int32, device="cuda"), 16)                  # nobody has a route
        check_order(torch.full((t, k), 7, dtype=torch.int32, device="cuda"), 16)                   # all to one expert, the same one twice in a token
        check_order(torch.full((t, k), 2 ** 31 - 1, dtype=torch.int32, device="cuda"), 1024)
        check_order(torch.full((t, k), -2 ** 31, dtype=torch.int32, device="cuda"), 1024)
    wide = make_ids(700, 12, 50, 3)
    check_order(wide[:, 2:9], 50)                                                                  # strided rows
    check_order(wide.t().contiguous().t()[:, :5], 50)                                              # columns first: a copy
    check_order(wide[:1].expand(300, -1), 50)


def rand(shape, kind, seed):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(kind)


def bits(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


@pytest.mark.parametrize("h", (1, 3, 8, 63, 64, 520, 2048, 7168))
@pytest.mark.parametrize("kind", (torch.int8, torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32, torch.int32))
def test_sort_copies(h, kind):
    for t, k, e, masked in ((1, 1, 4, 0.0), (37, 8, 16, 0.3), (700, 4, 8, 0.0)):
        x = (rand((t, h + 5), torch.float32, h) * 50).to(kind)
        order = ks.route_sort(make_ids(t, k, e, 1, masked), e)
        route = order.route_of_row.long()
        for v in (x[:, :h].contiguous(), x[:, 5:], x[:, 1:h + 1]):
            want = torch.where((route >= 0)[:, None], bits(v)[(route // k).clamp(min=0)], torch.zeros((), dtype=bits(v).dtype, device="cuda"))
            got = ks.sort_tokens(v, order)
            assert got.dtype == kind and torch.equal(bits(got), want)
        one = ks.sort_tokens(v[:, 0].contiguous(), order)
        assert one.shape == (t * k,) and torch.equal(bits(one), want[:, 0])


def unsort_exact(rows, order, w):
    """(sum in 64 bits, sum of absolute values)"""
    there = order.row_of >= 0
    picked = rows.double()[order.row_of.long().clamp(min=0)]
    picked = torch.where(there[..., None], picked, 0.0) * (1.0 if w is None else w.double()[..., None])
    return picked.sum(dim=1), picked.abs().sum(dim=1)


def close(got, exact, size, adds):
    """fp32 additions and products of `adds` terms of total size `size`, one rounding to the type."""
    tol = exact.abs() * torch.finfo(got.dtype).eps / 2 * (1 + 2.0 ** -10) + size * adds * 2.0 ** -24 * 1.1 + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    off = (got.double() - exact).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


@pytest.mark.parametrize("weighted", (True, False))
@pytest.mark.parametrize("h", (1, 7, 8, 100, 128, 2048, 7168))
@pytest.mark.parametrize("kind", KINDS)
def test_unsort_and_gradients(kind, h, weighted):
    kind = KINDS[kind]
    for t, k, e, masked in ((1, 1, 3, 0.0), (19, 8, 16, 0.4), (300, 5, 4, 0.1), (33, 17, 64, 0.5)):
        order = ks.route_sort(make_ids(t, k, e, h, masked), e)
        n = int(order.offsets[-1])
        rows = rand((t * k, h), kind, 1)
        rows[n:] = float("nan")                                    # behind the last segment: never read
        w = rand((t, k), torch.float32, 2) if weighted else None
        if weighted:
            w = torch.where(order.row_of >= 0, w, float("inf"))    # nor is the weight of a route that is none
        dy = rand((t, h), kind, 3)
        rows.requires_grad_()
        if weighted:
            w.requires_grad_()
        y = ks.unsort_tokens(rows, order, w)
        exact, size = unsort_exact(rows.detach(), order, None if w is None else torch.where(order.row_of >= 0, w.detach(), 0.0))
        close(y.detach(), exact, size, 2 * k)
        grads = torch.autograd.grad(y, (rows, w) if weighted else (rows,), dy)
        route = order.route_of_row.long()
        live = route[:n]
        want = dy.double()[live // k] * (w.detach().double().flatten()[live][:, None] if weighted else 1.0)
        close(grads[0][:n], want, want.abs(), 1)
        assert not bool(grads[0][n:].any())
        if weighted:
            prod = rows.detach()[:n].double() * dy.double()[live // k]
            dw = torch.zeros(t * k, dtype=torch.float64, device="cuda").index_copy_(0, live, prod.sum(dim=1))
            dabs = torch.zeros(t * k, dtype=torch.float64, device="cuda").index_copy_(0, live, prod.abs().sum(dim=1))
            close(grads[1].flatten(), dw, dabs, h + 1)
        # one of the two at a time: the same bits
        if weighted:
            for which in (0, 1):
                r2, w2 = rows.detach().requires_grad_(which == 0), w.detach().requires_grad_(which == 1)
                g, = torch.autograd.grad(ks.unsort_tokens(r2, order, w2), ((r2, w2)[which],), dy)
                assert torch.equal(g, grads[which])
        # the sorted rows' gradient: the sum over a token's rows
        x = rand((t, h), kind, 4).requires_grad_()
        g = rand((t * k, h), kind, 5)
        g[n:] = float("nan")
        dx, = torch.autograd.grad(ks.sort_tokens(x, order), x, g)
        close(dx, *unsort_exact(g, order, None), 2 * k)


def test_gradient_against_differences():
    """Central differences of a fp32 function of both operators, whose parts are linear in x and in the weights."""
    t, k, e, h = 6, 3, 4, 16
    order = ks.route_sort(make_ids(t, k, e, 5, 0.2), e)
    x, w, m, c = rand((t, h), torch.float32, 1), rand((t, k), torch.float32, 2), rand((t * k, h), torch.float32, 3), rand((t, h), torch.float32, 4)

    def f(x, w):
        return (ks.unsort_tokens(ks.sort_tokens(x, order) * m, order, w) * c).sum()

    xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(f(xr, wr), (xr, wr))
    for v, d, other in ((x, dx, "x"), (w, dw, "w")):
        for i in range(0, v.numel(), 5):
            up, down = v.clone(), v.clone()
            up.view(-1)[i] += 0.5
            down.view(-1)[i] -= 0.5
            diff = (f(up, w) - f(down, w)) if other == "x" else (f(x, up) - f(x, down))
            # f is linear in either: the difference is the gradient but for fp32 sums of a few hundred terms of size up to about 30
            assert abs(float(diff) - float(d.view(-1)[i])) < 2e-3


def test_strided_gradients_and_buffers():
    t, k, e, h = 50, 4, 8, 72
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    rows = rand((t * k, h + 9), torch.bfloat16, 1)[:, 4:h + 4].requires_grad_()
    w = rand((k, t), torch.float32, 2).t().requires_grad_()
    y = ks.unsort_tokens(rows, order, w)
    exact, size = unsort_exact(rows.detach(), order, w.detach())
    close(y.detach(), exact, size, 2 * k)
    for dy in (torch.ones((), dtype=torch.bfloat16, device="cuda").expand(t, h), rand((1, h), torch.bfloat16, 3).expand(t, h), rand((h, t), torch.bfloat16, 4).t()):
        got = torch.autograd.grad(y, (rows, w), dy, retain_graph=True)
        want = torch.autograd.grad(y, (rows, w), dy.contiguous(), retain_graph=True)
        assert torch.equal(got[0], want[0])
        close(got[1].flatten(), want[1].double().flatten(), want[1].double().abs().flatten() + 100.0, h)     # other pieces per thread: another order


def test_captured_training_step():
    """Forward and backward in one graph, of leaves made inside it, while an eager graph of the same tensors lives; replayed on other routes."""
    t, k, e, h = 200, 4, 16, 256
    ids, x, w, dy = make_ids(t, k, e, 1), rand((t, h), torch.bfloat16, 1), rand((t, k), torch.float32, 2), rand((t, h), torch.bfloat16, 3)

    def step():
        xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
        order = ks.route_sort(ids, e)
        y = ks.unsort_tokens(ks.sort_tokens(xl, order), order, wl)
        return (y.detach(), *torch.autograd.grad(y, (xl, wl), dy))

    alive = ks.unsort_tokens(ks.sort_tokens(x.detach().requires_grad_(), ks.route_sort(ids, e)), ks.route_sort(ids, e))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2, 3):
        ids.copy_(make_ids(t, k, e, seed))
        x.copy_(rand((t, h), torch.bfloat16, seed + 10))
        graph.replay()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
    assert alive.shape == (t, h)


def test_capture_beside_a_live_graph_is_refused():
    """A captured backward pass of leaves whose eager graph lives would end the process: the forward call says so instead."""
    t, k, e, h = 20, 2, 4, 64
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    x, w = rand((t, h), torch.bfloat16, 1).requires_grad_(), rand((t, k), torch.float32, 2).requires_grad_()
    alive = ks.unsort_tokens(ks.sort_tokens(x, order), order, w)
    rows = rand((t * k, h), torch.bfloat16, 3)
    said = []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows.mul_(1.0)
        for call in (lambda: ks.sort_tokens(x, order), lambda: ks.unsort_tokens(rows, order, w)):
            try:
                call()
            except ValueError as exc:
                said.append(str(exc))
    assert len(said) == 2 and all("alive" in s for s in said)
    assert alive.shape == (t, h)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):                                  # the graph is gone, and its nodes with it
        y = ks.unsort_tokens(ks.sort_tokens(x, order), order, w).detach()
    graph.replay()
    with torch.no_grad():
        assert torch.equal(y, ks.unsort_tokens(ks.sort_tokens(x, order), order, w))


def test_capture_beside_a_live_graph_of_an_input_is_refused():
    """The same where the leaf is behind an operation of the capture, or the whole input was made outside it."""
    t, k, e, h = 20, 2, 4, 64
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    x, w = rand((t, h), torch.bfloat16, 1).requires_grad_(), rand((t, k), torch.float32, 2).requires_grad_()
    rows = rand((t * k, h), torch.bfloat16, 3)
    alive = x * 2
    said = []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: ks.sort_tokens(x + 1, order), lambda: ks.sort_tokens(alive, order), lambda: ks.unsort_tokens(rows, order, w * w)):
            try:
                call()
            except ValueError as exc:
                said.append(str(exc))
    assert len(said) == 2 and all("alive" in s for s in said)      # w has no graph outside


def test_capture_on_two_streams():
    """A stream that joined the capture is part of it: its nodes refuse nothing, and the gradients are those of eager calls."""
    t, k, e, h = 20, 2, 4, 64
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    x, g = rand((t, h), torch.float32, 1).requires_grad_(), rand((t * k, h), torch.float32, 3)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            twice = x * 2
        torch.cuda.current_stream().wait_stream(side)
        dx, = torch.autograd.grad(ks.sort_tokens(twice, order), x, g)
    graph.replay()
    eager, = torch.autograd.grad(ks.sort_tokens(x * 2, order), x, g)
    assert torch.equal(dx, eager)


def test_gradients_of_gradients_are_refused():
    t, k, e, h = 6, 2, 4, 16
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    x, w = rand((t, h), torch.float32, 1).requires_grad_(), rand((t, k), torch.float32, 2).requires_grad_()
    y = ks.unsort_tokens(ks.sort_tokens(x, order), order, w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w), create_graph=True)
    for d in (dx, dw):
        with pytest.raises(RuntimeError):
            d.sum().backward(retain_graph=True)


def test_backward_accumulates():
    """.backward() twice, of a scale column as well: gradients add up in .grad."""
    t, k, e = 40, 3, 8
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    s, m = rand((t,), torch.float32, 1).requires_grad_(), rand((t * k,), torch.float32, 2)
    for _ in range(2):
        (ks.sort_tokens(s, order) * m).sum().backward()
    exact, size = unsort_exact(m[:, None], order, None)
    close(s.grad, 2 * exact[:, 0], 2 * size[:, 0], 2 * k)


def test_empty_batch():
    order = ks.route_sort(torch.empty(0, 4, dtype=torch.int32, device="cuda"), 8)
    assert order.offsets.tolist() == [0] * 9
    x = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    rows = ks.sort_tokens(x, order)
    w = torch.empty(0, 4, device="cuda", requires_grad=True)
    y = ks.unsort_tokens(rows, order, w)
    assert rows.shape == (0, 64) and y.shape == (0, 64)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape


@pytest.mark.parametrize("t,h", [(1 << 16, 265), (66_000_000, 265)])
def test_unsort_of_one_row_for_all(t, h):
    """A row that every token has; 66 million of 33 vectors and an element are more than a grid's threads (35 GB of output)."""
    if t * h * 2.4 > torch.cuda.mem_get_info()[0] + torch.cuda.memory_reserved() - torch.cuda.memory_allocated():
        pytest.skip("not enough device memory")
    x = torch.randint(-127, 128, (1, h), device="cuda").to(torch.bfloat16)
    order = ks.route_sort(torch.zeros(t, 1, device="cuda", dtype=torch.int32), 1)
    y = ks.unsort_tokens(x.expand(t, -1), order)
    for part in y.split(1 << 20):
        assert bool((part == x).all())


def test_rows_behind_2_31_elements():
    """2^21 rows of 1032: element offsets pass 2^31."""
    t, k, e, h = 1 << 19, 4, 8, 1032
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, e, (t, k), generator=g, device="cuda", dtype=torch.int32)
    order = ks.route_sort(ids, e)
    x = torch.randint(-127, 128, (t, h), generator=g, device="cuda", dtype=torch.int8)
    rows = ks.sort_tokens(x, order)
    at = torch.tensor([0, 1, t * k // 2, t * k - 2, t * k - 1], device="cuda")
    assert torch.equal(rows[at], x[order.route_of_row[at].long() // k])
    wide = rows.to(torch.bfloat16)
    y = ks.unsort_tokens(wide, order, torch.full((t, k), 0.25, device="cuda"))
    assert torch.equal(y, x.to(torch.bfloat16))


def test_function_transforms_and_tangents_raise():
    """What the calls have no rule for is an error, not a derivative of zero."""
    import torch.autograd.forward_ad as forward_ad
    t, k, e, h = 12, 2, 4, 32
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    x, w, rows = rand((t, h), torch.float32, 1), rand((t, k), torch.float32, 2), rand((t * k, h), torch.float32, 3)
    for f, args in ((lambda v: ks.sort_tokens(v, order), (x,)), (lambda v, u: ks.unsort_tokens(v, order, u), (rows, w))):
        ones = tuple(torch.ones_like(v) for v in args)
        for transform in (lambda: torch.func.jvp(f, args, ones), lambda: torch.func.grad(lambda *v: f(*v).sum())(*args), lambda: torch.func.vmap(f)(*(v[None] for v in args))):
            with pytest.raises((RuntimeError, ValueError)):
                transform()
        for i in range(len(args)):
            with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
                f(*(forward_ad.make_dual(v, o) if j == i else v for j, (v, o) in enumerate(zip(args, ones))))


def test_unsort_keeps_only_what_its_gradient_reads():
    """The rows are read for the weights' gradient, the weights for the rows': what is not read may change before the backward pass, and goes with its
    last reference."""
    t, k, e, h = 64, 4, 8, 1024
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    leaf, w, dy = rand((t * k, h), torch.bfloat16, 1).requires_grad_(), rand((t, k), torch.float32, 2), rand((t, h), torch.bfloat16, 3)
    wl = w.clone().requires_grad_()
    want_rows, want_w = torch.autograd.grad(ks.unsort_tokens(leaf, order, wl), (leaf, wl), dy)
    plain, = torch.autograd.grad(ks.unsort_tokens(leaf, order), leaf, dy)
    for weights, want in ((w, want_rows), (None, plain)):
        rows = leaf * 1
        y = ks.unsort_tokens(rows, order, weights)
        rows.mul_(2)                                               # not read: no error, and the derivative of `rows` as it was
        got, = torch.autograd.grad(y, leaf, dy)
        assert torch.equal(got, want)
        rows = leaf * 1
        y = ks.unsort_tokens(rows, order, weights)
        held = torch.cuda.memory_allocated()
        del rows
        assert held - torch.cuda.memory_allocated() >= t * k * h * 2
        assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want)
    # the weights' gradient alone: the rows are read, the weights are not
    weights = wl * 1
    y = ks.unsort_tokens(leaf.detach(), order, weights)
    weights.mul_(2)
    assert torch.equal(torch.autograd.grad(y, wl, dy)[0], want_w)
    rows = leaf.detach().clone()
    y = ks.unsort_tokens(rows, order, wl)
    rows.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, wl, dy)
    # odd widths as well, where a row's phase is worked out from its address
    for h in (7, 33, 1025):
        odd, dy = rand((t * k, h), torch.float16, 4).requires_grad_(), rand((t, h), torch.float16, 5)
        both = torch.autograd.grad(ks.unsort_tokens(odd, order, wl), (odd, wl), dy)
        assert torch.equal(torch.autograd.grad(ks.unsort_tokens(odd, order, w), odd, dy)[0], both[0])
        assert torch.equal(torch.autograd.grad(ks.unsort_tokens(odd.detach(), order, wl), wl, dy)[0], both[1])


def test_capture_beside_a_live_graph_of_a_side_stream():
    """A stream other than the default one joins a capture when the backward pass reaches its nodes: a leaf whose live graph was built there is taken."""
    t, k, e, h = 20, 2, 4, 64
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    x, w = rand((t, h), torch.float32, 1).requires_grad_(), rand((t, k), torch.float32, 2).requires_grad_()
    g, dy = rand((t * k, h), torch.float32, 3), rand((t, h), torch.float32, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive, other = x * 2, w * 2
    torch.cuda.synchronize()

    def grads(inputs):
        v, u = inputs()
        return (torch.autograd.grad((ks.sort_tokens(v, order) * g).sum(), x, retain_graph=True)[0],
                torch.autograd.grad(ks.unsort_tokens(g, order, u), w, dy, retain_graph=True)[0])

    for inputs in (lambda: (x, w), lambda: (x + 1, w * w), lambda: (alive, other)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = grads(inputs)
        graph.replay()
        for got, want in zip(captured, grads(inputs)):
            assert torch.equal(got, want)
    # .backward() into .grad
    x.grad = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (ks.sort_tokens(x, order) * g).sum().backward()
    graph.replay()
    assert torch.equal(x.grad, torch.autograd.grad((ks.sort_tokens(x, order) * g).sum(), x)[0])


def test_a_gradient_with_a_tangent_is_refused():
    """Forward mode over a backward pass: the gradient that comes in carries a tangent though no input does."""
    import torch.autograd.forward_ad as forward_ad
    t, k, e, h = 12, 2, 4, 32
    order = ks.route_sort(make_ids(t, k, e, 1), e)
    x, w, rows = (v.requires_grad_() for v in (rand((t, h), torch.float32, 1), rand((t, k), torch.float32, 2), rand((t * k, h), torch.float32, 3)))
    for y, leaves in ((ks.sort_tokens(x, order), (x,)), (ks.unsort_tokens(rows, order, w), (rows, w)), (ks.unsort_tokens(rows, order), (rows,))):
        with forward_ad.dual_level():
            c = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises((RuntimeError, ValueError), match="forward-mode"):
                torch.autograd.grad((y * c).sum(), leaves, retain_graph=True)
        for g in torch.autograd.grad(y.sum(), leaves):             # and the call is one like any other without it
            assert bool(g.isfinite().all())
