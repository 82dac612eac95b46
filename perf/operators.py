"""Timed cases of the 8-bit operators and of the routing operators that have a gradient: root-mean-square norm and SwiGLU with an 8-bit
output and one scale per row, the 8-bit product with scales per token and channel (dense, and over the experts' segments of sorted
rows), and tokens sorted by expert and back.

`listed()` gives the named cases, `draw(rng)` one more of the same ranges. `run` computes a case in elementary torch operations, or with
`own` through the library's entry points; `exact` gives its outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EIGHT = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------------ cases
def _norm(t, h, kind="bf16", to="int8", residual=True, normed=False):
    return dict(op="norm", t=t, h=h, kind=kind, to=to, residual=residual, normed=normed)


def _swiglu(r, i, kind="bf16", to="int8"):
    return dict(op="swiglu", r=r, i=i, kind=kind, to=to)


def _mm(m, n, k, kind="int8", to="bf16"):
    return dict(op="mm", m=m, n=n, k=k, kind=kind, to=to)


def _grouped(t, k_top, e, n, k, kind="int8", to="bf16", masked=False):
    return dict(op="grouped", t=t, k_top=k_top, e=e, n=n, k=k, kind=kind, to=to, masked=masked)


def _order(t, k_top, e, h, kind="bf16", train=True, masked=False):
    return dict(op="order", t=t, k_top=k_top, e=e, h=h, kind=kind, train=train, masked=masked)


def listed():
    return [
        # the norm in front of a layer, one token being generated
        dict(_norm(1, 2048, to="e4m3"), name="norm_1_token"),
        # the same for a prompt, residual stream updated
        dict(_norm(8192, 7168, to="e4m3"), name="norm_prompt"),
        # a ragged chunk in fp16 whose normed rows the router reads as well
        dict(_norm(1777, 2047, kind="fp16", normed=True, residual=False), name="norm_chunk_odd_width"),
        # between an expert's two products, all routed rows of a prompt
        dict(_swiglu(65536, 768, to="e4m3"), name="swiglu_prompt"),
        # the same for a small batch
        dict(_swiglu(129, 2048, to="int8"), name="swiglu_129_rows"),
        # a linear layer, one token: a stream over the weights
        dict(_mm(1, 4096, 7168), name="mm_1_token"),
        # a small batch and a width that no tile divides, in e4m3
        dict(_mm(100, 2113, 7168, kind="e4m3", to="fp16"), name="mm_100_rows_odd_width"),
        # a prompt, bound by the tensor cores
        dict(_mm(8192, 4096, 12288), name="mm_prompt"),
        # experts' first product while a small batch generates: most of the weights for few rows each
        dict(_grouped(64, 8, 128, 1536, 2048), name="experts_64_tokens"),
        # and for a prompt, with uneven segments
        dict(_grouped(8192, 8, 128, 1536, 2048, kind="e4m3"), name="experts_prompt"),
        # tokens to the experts' order and back in a training step, with the gradients of both
        dict(_order(8192, 8, 128, 2048), name="order_train"),
        # the same in serving, 8-bit rows with their scales out and bf16 rows back; some routes belong to other ranks
        dict(_order(32, 8, 256, 7168, train=False, masked=True), name="order_32_tokens"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(("norm", "swiglu", "mm", "mm", "grouped", "grouped", "order"))
    kind, to = rng.choice(tuple(DTYPES)), rng.choice(tuple(EIGHT))
    if op == "norm":
        h = _log(rng, 64, 8192)
        return _norm(_log(rng, 1, min(32768, 8192 * 7168 // (2 * h))), h, kind, to, rng.random() < 0.7, rng.random() < 0.3)
    if op == "swiglu":
        i = _log(rng, 32, 4096)
        return _swiglu(_log(rng, 1, min(65536, 65536 * 768 // (2 * i))), i, kind, to)
    if op == "mm":
        n, k = _log(rng, 64, 8192), 16 * _log(rng, 4, 768)
        return _mm(_log(rng, 1, 8192), n, k, to, kind)
    if op == "grouped":
        e = _log(rng, 2, 128)
        return _grouped(_log(rng, 1, 4096), rng.randint(1, min(e, 8)), e, _log(rng, 64, 2048), 16 * _log(rng, 8, 128), to, kind, rng.random() < 0.3)
    e, h = _log(rng, 2, 256), _log(rng, 64, 7168)
    k_top = rng.randint(1, min(e, 8))
    return _order(_log(rng, 1, min(16384, 8192 * 8 * 2048 // (2 * h * k_top))), k_top, e, h, kind, rng.random() < 0.6, rng.random() < 0.3)


# ------------------------------------------------------------------------------------------------------------------ inputs
def _rows8(x, kind):
    """Rows in 8 bits and their scales, as a quantiser in front of the product leaves them."""
    dtype, top = EIGHT[kind]
    s = x.abs().amax(dim=-1, keepdim=True) / top
    q = (x / s).round().to(dtype) if kind == "int8" else (x / s).to(dtype)
    return q, s.squeeze(-1)


def _ids(case, gen):
    """Distinct experts per token, drawn with uneven popularity; where masked, routes of other ranks are out of range or -1."""
    t, e, k = case["t"], case["e"], case["k_top"]
    bias = torch.randn(e, generator=gen, device="cuda") * 0.6
    ids = (torch.randn(t, e, generator=gen, device="cuda") + bias).topk(k, dim=1).indices.int()
    if case["masked"]:
        u = torch.rand(t, k, generator=gen, device="cuda")
        ids = torch.where(u < 0.3, torch.full_like(ids, -1), torch.where(u > 0.9, ids + e, ids))
    return ids


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    op, s = case["op"], dict(case=case)
    if op == "norm":
        kind = DTYPES[case["kind"]]
        channel = 1.0 + 3.0 * (torch.rand(case["h"], generator=gen, device="cuda") < 0.01)      # a few channels are larger than the others
        s["x"] = randn(case["t"], case["h"]).to(kind)
        s["residual"] = (randn(case["t"], case["h"]) * channel * 2).to(kind) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * randn(case["h"])).to(kind)
    elif op == "swiglu":
        s["x"] = (randn(case["r"], 2 * case["i"]) * 1.5).to(DTYPES[case["kind"]])
    elif op == "mm":
        s["a"], s["a_scale"] = _rows8(randn(case["m"], case["k"]), case["kind"])
        s["b"], s["b_scale"] = _rows8(randn(case["n"], case["k"]) * 0.02, case["kind"])
    elif op == "grouped":
        e = case["e"]
        flat = _ids(case, gen).flatten()
        counts = torch.bincount(flat[(flat >= 0) & (flat < e)], minlength=e)
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
        s["most"] = int(counts.max())
        s["a"], s["a_scale"] = _rows8(randn(flat.numel(), case["k"]), case["kind"])
        s["b"], s["b_scale"] = _rows8(randn(e, case["n"], case["k"]) * 0.02, case["kind"])
    else:
        kind = DTYPES[case["kind"]]
        t, k, h = case["t"], case["k_top"], case["h"]
        s["ids"] = _ids(case, gen)
        s["weights"] = randn(t, k).softmax(dim=1)
        x, s["products"] = randn(t, h), randn(t * k, h).to(kind)      # products: what the experts made of the sorted rows
        if case["train"]:
            s["x"], s["dy"], s["drows"] = x.to(kind), randn(t, h).to(kind), randn(t * k, h).to(kind)
        else:
            s["x"], s["scale"] = _rows8(x, "int8")
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _quantised(y, to):
    """(values in 8 bits, scales) of fp32 rows."""
    dtype, top = EIGHT[to]
    scale = y.abs().amax(dim=1) / top
    z = torch.where(scale[:, None] > 0, y / scale[:, None], torch.zeros_like(y)).clamp(-top, top)
    return (z.round() if to == "int8" else z).to(dtype), scale


def _values(q, scale):
    """int8 rows as the values they stand for, in 16 bits; e4m3 codes are values already, beside their scales."""
    return torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)) if q.dtype == torch.int8 else q


def _plain_norm(s):
    x, case = s["x"], s["case"]
    h = x.float() if s["residual"] is None else x.float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
    q, scale = _quantised(y, case["to"])
    return q, scale, h.to(x.dtype), y.to(x.dtype) if case["normed"] else None


def _plain_swiglu(s):
    g, u = s["x"].float().chunk(2, dim=1)
    return _quantised(g / (1.0 + torch.exp(-g)) * u, s["case"]["to"])


def _plain_mm(s):
    # in 64 bits: sums of int8 products pass 2^24
    acc = s["a"].double() @ s["b"].double().t()
    return (acc * s["a_scale"].double()[:, None] * s["b_scale"].double()).to(DTYPES[s["case"]["to"]])


def _plain_grouped(s):
    # every expert's rows padded to the largest segment; places past a segment read row 0 and are not written
    a, offsets, most = s["a"], s["offsets"].long(), s["most"]
    place = torch.arange(most, device=a.device)
    row = offsets[:-1, None] + place
    live = row < offsets[1:, None]
    rows = a.float()[torch.where(live, row, 0)]
    acc = torch.bmm(rows.double(), s["b"].double().transpose(1, 2))
    acc = acc * s["a_scale"].double()[torch.where(live, row, 0)][:, :, None] * s["b_scale"].double()[:, None, :]
    out = torch.zeros((a.shape[0] + 1, s["b"].shape[1]), dtype=DTYPES[s["case"]["to"]], device=a.device)
    out.index_copy_(0, torch.where(live, row, a.shape[0]).flatten(), acc.to(out.dtype).flatten(0, 1))
    return out[:-1]


def _plain_sort(ids, e):
    flat = ids.flatten().long()
    valid = (flat >= 0) & (flat < e)
    key = torch.where(valid, flat, e)
    by = torch.argsort(key, stable=True)
    counts = torch.zeros(e + 1, dtype=torch.int64, device=ids.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([counts.new_zeros(1), counts[:e].cumsum(0)])
    row = torch.arange(flat.numel(), device=ids.device)
    row_of = torch.empty_like(row).scatter_(0, by, row)
    row_of = torch.where(valid, row_of, -1).view(ids.shape)
    return offsets.int(), row_of.int(), torch.where(row < offsets[-1], by, -1).int()


def _plain_take(x, route_of_row, k):
    """x[token of each row], zero behind the last valid row."""
    token = torch.div(route_of_row.long(), k, rounding_mode="floor")
    picked = x[token.clamp(min=0)]
    live = (route_of_row >= 0).view(-1, *[1] * (picked.dim() - 1))
    return torch.where(live, picked, torch.zeros((), dtype=picked.dtype, device=picked.device)) if picked.dtype != torch.int8 else picked * live


def _plain_order(s):
    case, ids, w = s["case"], s["ids"], s["weights"]
    k, kind = case["k_top"], DTYPES[case["kind"]]
    offsets, row_of, route_of_row = _plain_sort(ids, case["e"])
    at, there = row_of.long().clamp(min=0), (row_of >= 0)
    rows = _plain_take(s["x"], route_of_row, k)
    zero = torch.zeros((), device=ids.device)
    slots = torch.where(there[..., None], s["products"][at].float(), zero)
    out = dict(offsets=offsets, row_of=row_of, rows=rows, y=(w[..., None] * slots).sum(dim=1).to(kind))
    if not case["train"]:
        return dict(out, scales=_plain_take(s["scale"], route_of_row, k))
    dy = s["dy"].float()
    dproducts = _plain_take((w[..., None] * dy[:, None, :]).flatten(0, 1), route_of_row, 1)
    dslots = torch.where(there[..., None], s["drows"][at].float(), zero)
    return dict(out, dweights=(slots * dy[:, None, :]).sum(dim=2), dproducts=dproducts.to(kind), dx=dslots.sum(dim=1).to(kind))


# ------------------------------------------------------------------------------------------------------------------ the library's calls
def _own_order(s):
    import kernelschema_b200 as ks
    case = s["case"]
    if not case["train"]:
        order = ks.route_sort(s["ids"], case["e"])
        return dict(offsets=order.offsets, row_of=order.row_of, rows=ks.sort_tokens(s["x"], order), scales=ks.sort_tokens(s["scale"], order),
                    y=ks.unsort_tokens(s["products"], order, s["weights"]))
    x, products, w = (s[name].detach().requires_grad_() for name in ("x", "products", "weights"))
    order = ks.route_sort(s["ids"], case["e"])
    rows = ks.sort_tokens(x, order)
    y = ks.unsort_tokens(products, order, w)
    dx, dproducts, dw = torch.autograd.grad((rows, y), (x, products, w), (s["drows"], s["dy"]))
    return dict(offsets=order.offsets, row_of=order.row_of, rows=rows, y=y, dweights=dw, dproducts=dproducts, dx=dx)


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        import kernelschema_b200 as ks
        if op == "norm":
            q, scale, hidden, normed = ks.rmsnorm_quantize(state["x"], state["weight"], state["residual"], EPS, EIGHT[case["to"]][0], case["normed"])
        elif op == "swiglu":
            q, scale = ks.swiglu_quantize(state["x"], EIGHT[case["to"]][0])
        elif op == "mm":
            return ks.mm_8bit(state["a"], state["a_scale"], state["b"], state["b_scale"], out_dtype=DTYPES[case["to"]])
        elif op == "grouped":
            return ks.mm_8bit_grouped(state["a"], state["a_scale"], state["b"], state["b_scale"], state["offsets"], out_dtype=DTYPES[case["to"]])
        else:
            return _own_order(state)
    elif op == "norm":
        q, scale, hidden, normed = _plain_norm(state)
    elif op == "swiglu":
        q, scale = _plain_swiglu(state)
    else:
        return {"mm": _plain_mm, "grouped": _plain_grouped, "order": _plain_order}[op](state)
    if op == "swiglu":
        return dict(values=_values(q, scale), scale=scale)
    return dict(values=_values(q, scale), scale=scale, hidden=hidden if case["residual"] else None, normed=normed)


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def _exact_rows8(y, to):
    dtype, top = EIGHT[to]
    peak = y.abs().max(dim=1).values
    code = y * (top / peak)[:, None]
    if to == "int8":
        return torch.round(code) * (peak / top)[:, None], peak / top
    step = torch.exp2(torch.floor(torch.log2(code.abs().clamp(min=2.0 ** -6))) - 3)      # e4m3: three fraction bits, least exponent -6
    return torch.round(code / step) * step, peak / top


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double()
        if case["residual"]:
            h += s["residual"].double()
        y = h * s["weight"].double() / torch.sqrt(torch.linalg.vecdot(h, h) / case["h"] + EPS)[:, None]
        q, scale = _exact_rows8(y, case["to"])
        return dict(values=q, scale=scale, hidden=h if case["residual"] else None, normed=y if case["normed"] else None)
    if op == "swiglu":
        g, u = s["x"][:, :case["i"]].double(), s["x"][:, case["i"]:].double()
        q, scale = _exact_rows8(u * g * torch.sigmoid(g), case["to"])
        return dict(values=q, scale=scale)
    if op == "mm":
        a, out = s["a"].double() * s["a_scale"].double()[:, None], []
        for b, c in zip(s["b"].split(1024), s["b_scale"].split(1024)):
            out.append(torch.einsum("mk,nk->mn", a, b.double() * c.double()[:, None]))
        return torch.cat(out, dim=1)
    if op == "grouped":
        at, out = s["offsets"].tolist(), torch.zeros(s["a"].shape[0], case["n"], dtype=torch.float64, device="cuda")
        for e in range(case["e"]):
            if at[e] < at[e + 1]:
                a = s["a"][at[e]:at[e + 1]].double() * s["a_scale"][at[e]:at[e + 1]].double()[:, None]
                out[at[e]:at[e + 1]] = a @ (s["b"][e].double() * s["b_scale"][e].double()[:, None]).t()
        return out
    # routes of expert 0 in the order of their tokens, then those of expert 1, ...
    t, k, h = case["t"], case["k_top"], case["h"]
    ids, w = s["ids"].flatten().cpu().numpy(), s["weights"].double().flatten()
    order = [int(r) for e in range(case["e"]) for r in (ids == e).nonzero()[0]]
    route = torch.tensor(order, dtype=torch.int64, device="cuda")
    token, n = route // k, len(order)
    products = s["products"][:n].double()
    y = torch.zeros(t, h, dtype=torch.float64, device="cuda").index_add_(0, token, products * w[route][:, None])
    out = dict(offsets=None, row_of=None, rows=None, y=y)
    if not case["train"]:
        return dict(out, scales=None)
    dy = s["dy"].double()
    dx = torch.zeros_like(y).index_add_(0, token, s["drows"][:n].double())
    dproducts = torch.zeros(t * k, h, dtype=torch.float64, device="cuda")
    dproducts[:n] = dy[token] * w[route][:, None]
    dweights = torch.zeros(t * k, dtype=torch.float64, device="cuda")
    dweights[route] = (products * dy[token]).sum(dim=1)
    return dict(out, dx=dx, dweights=dweights.view(t, k), dproducts=dproducts)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    op, size = case["op"], {"bf16": 2, "fp16": 2, "fp32": 4}
    if op == "norm":
        t, h, b = case["t"], case["h"], size[case["kind"]]
        return dict(bytes=t * h * (b * (1 + 2 * case["residual"] + case["normed"]) + 1) + 4 * t + h * b, flops=6 * t * h)
    if op == "swiglu":
        r, i = case["r"], case["i"]
        return dict(bytes=r * i * (2 * size[case["kind"]] + 1) + 4 * r, flops=8 * r * i)
    if op == "mm":
        m, n, k = case["m"], case["n"], case["k"]
        return dict(bytes=m * k + n * k + 4 * (m + n) + m * n * size[case["to"]], flops=2 * m * n * k)
    held = 0.6 if case["masked"] else 1.0
    rows = case["t"] * case["k_top"]
    if op == "grouped":
        n, k, e = case["n"], case["k"], case["e"]
        busy = e * (1.0 - (1.0 - case["k_top"] * held / e) ** case["t"])      # experts that have rows, were all equally popular
        return dict(bytes=rows * held * k + busy * n * k + 4 * (rows + e * n) + rows * n * size[case["to"]], flops=2 * rows * held * n * k)
    t, h, b = case["t"], case["h"], size[case["kind"]]
    ints = 4 * (3 * rows + case["e"] + 1 + rows)
    if not case["train"]:
        return dict(bytes=ints + t * h + rows * h + rows * held * h * b + t * h * b, flops=2 * rows * held * h)
    # in: x, products, dy and the sorted rows' gradient; out: rows, y and the gradients of products and x
    return dict(bytes=ints + 4 * rows + h * b * (4 * t + 2 * rows * (1 + held)), flops=6 * rows * held * h)
