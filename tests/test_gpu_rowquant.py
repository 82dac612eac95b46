"""RMS norm and SwiGLU with an 8-bit output against their definitions in 64 bits."""
import pytest
import torch

import kernelschema_b200 as ks

pytestmark = pytest.mark.gpu

KINDS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
#: fp32 chains of a few hundred additions in a tree and a handful of products: far below 64 roundings of 2^-24
REL = 64 * 2.0 ** -24


def check_codes(q, scale, y, dtype):
    """q and scale against the exact row y: the scale to fp32 accuracy, each code within half a step of y / scale (and what fp32 arithmetic adds)."""
    top = TOP[dtype]
    amax = y.abs().amax(dim=1)
    assert q.dtype == dtype and scale.dtype == torch.float32
    torch.testing.assert_close(scale.double(), amax / top, rtol=REL, atol=0)
    code = torch.where(amax[:, None] > 0, y * (top / amax)[:, None], torch.zeros_like(y))
    if dtype == torch.int8:
        half = torch.full_like(code, 0.5)
        assert int(q.int().abs().max()) <= 127
    else:
        half = torch.exp2(torch.floor(torch.log2(code.abs().clamp(min=2.0 ** -6))) - 4)
    # fp32 arithmetic moves a code by REL of its size (of the row's size where terms cancel, which they do not here: y is a product)
    off = (q.double() - code).abs()
    assert bool((off <= half * (1 + 1e-6) + REL * code.abs() + (0 if dtype == torch.int8 else 2.0 ** -10 * REL)).all()), float((off - half).max())


def norm_exact(x, w, residual, eps):
    h = x.double() if residual is None else x.double() + residual.double()
    return h, h * (h.square().mean(dim=1, keepdim=True) + eps) ** -0.5 * w.double()


def rows(t, h, kind, seed, scale=1.0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(t, h + pad, generator=g, device="cuda") * scale).to(kind)[:, :h]


def half_step(kind):
    return torch.finfo(kind).eps / 2


# widths of one vector, of a warp's and a block's rows, at the borders between the forms and off every vector; up to the largest
WIDTHS = (1, 7, 8, 64, 130, 256, 257, 512, 1016, 1024, 1032, 2047, 4096, 7168, 8200, 16384, 32767, 32768)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TOP)
@pytest.mark.parametrize("h", WIDTHS)
def test_norm(h, dtype, kind):
    kind = KINDS[kind]
    for t, residual, normed, wide in ((1, True, True, False), (3, False, True, True), (331, True, False, False)):
        if t * h > 4_000_000:
            t = 5
        x, r = rows(t, h, kind, h), (rows(t, h, kind, h + 1, 2.0) if residual else None)
        w = (1 + 0.1 * rows(1, h, torch.float32, 7)[0]).to(torch.float32 if wide else kind)
        q, scale, hidden, n = ks.rmsnorm_quantize(x, w, r, 1e-5, dtype, normed)
        he, y = norm_exact(x, w, r, 1e-5)
        check_codes(q, scale, y, dtype)
        if residual:
            assert torch.equal(hidden, (x.float() + r.float()).to(kind))
        else:
            assert hidden is x
        if normed:
            assert bool(((n.double() - y).abs() <= (half_step(kind) * (1 + 1e-6) + REL) * y.abs() + torch.finfo(kind).smallest_normal * 2.0 ** -7).all())
        else:
            assert n is None


@pytest.mark.parametrize("rows_n", (1, 295, 296, 1000))
def test_norm_of_few_and_many_rows_agrees(rows_n):
    """The forms of a block (few rows: more threads) give codes of the same values."""
    x, w = rows(rows_n, 4096, torch.bfloat16, 3), rows(1, 4096, torch.bfloat16, 4)[0]
    q, s, _, _ = ks.rmsnorm_quantize(x, w, dtype=torch.float8_e4m3fn)
    check_codes(q, s, norm_exact(x, w, None, 1e-6)[1], torch.float8_e4m3fn)


@pytest.mark.parametrize("h,pad", ((512, 8), (512, 3), (513, 5), (4096, 16), (2048, 1)))
def test_norm_strided_rows_and_buffers(h, pad):
    t, kind = 37, torch.bfloat16
    x, r, w = rows(t, h, kind, 1, pad=pad), rows(t, h, kind, 2, pad=pad), rows(1, h, kind, 3)[0]
    he, y = norm_exact(x, w, r, 1e-6)
    wide = [torch.full((t, h + pad), -17, dtype=d, device="cuda") for d in (torch.int8, kind, kind)]
    scale = torch.empty(t, device="cuda")
    got = ks.rmsnorm_quantize(x, w, r, out=(wide[0][:, :h], scale, wide[1][:, :h], wide[2][:, :h]))
    check_codes(got[0], got[1], y, torch.int8)
    assert torch.equal(got[2], he.float().to(kind))          # a sum of two bf16 values of like size is exact in fp32
    assert bool(((got[3].double() - y).abs() <= (half_step(kind) * (1 + 1e-6) + REL) * y.abs() + 1e-38).all())
    for b in wide:
        assert bool((b[:, h:] == -17).all())


def test_norm_in_place_and_repeated_row():
    x, r, w = rows(300, 2048, torch.float16, 1), rows(300, 2048, torch.float16, 2), rows(1, 2048, torch.float16, 3)[0]
    want = ks.rmsnorm_quantize(x, w, r)
    for target in (0, 1):
        a, b = x.clone(), r.clone()
        got = ks.rmsnorm_quantize(a, w, b, out=(None, None, (a, b)[target], None))
        assert got[2] is (a, b)[target]
        for u, v in zip(got[:3], want[:3]):
            assert torch.equal(u, v)
        assert torch.equal((b, a)[target], (r, x)[target])
    one = x[:1].expand(40, -1)                               # row stride 0
    q, s, _, _ = ks.rmsnorm_quantize(one, w)
    assert torch.equal(q, q[:1].expand(40, -1)) and torch.equal(s, s[:1].expand(40))
    t = ks.rmsnorm_quantize(x.t().contiguous().t(), w, r)     # columns first: read as a copy
    assert torch.equal(t[0], want[0])


@pytest.mark.parametrize("dtype", TOP)
@pytest.mark.parametrize("h", (96, 4096, 1025))
def test_special_rows(h, dtype):
    x = rows(12, h, torch.float32, 5)
    w = torch.ones(h, device="cuda")
    x[1] = 0
    x[2, h // 2] = float("nan")
    x[3, h - 1] = float("inf")
    x[4, 0] = float("-inf")
    x[5] *= 1e30                                             # the squares' sum leaves fp32
    x[6] = 0
    x[6, 3] = 1e-30                                          # with eps below: y of 1e-30 / 1e-3, above the least amax
    x[7] = 0
    x[7, 3] = 1e-39                                          # y of 1e-36: counts as zero
    q, s, _, n = ks.rmsnorm_quantize(x, w, None, 1e-6, dtype, True)
    for bad in (2, 3, 4, 5):
        assert bool(s[bad].isnan()) and not bool(q[bad].float().any()), bad
    assert bool(n[5].isnan().all()) and bool(n[2].isnan().all())
    for zero in (1, 7):
        assert float(s[zero]) == 0 and not bool(q[zero].float().any())
    assert float(q[6, 3].float()) == TOP[dtype] and int((q[6].float() != 0).sum()) == 1
    good = [0, 8, 9, 10, 11]
    check_codes(q[good], s[good], norm_exact(x[good], w, None, 1e-6)[1], dtype)
    q, s, _, _ = ks.rmsnorm_quantize(x[:1], torch.full((h,), float("nan"), device="cuda"), None, 1e-6, dtype)
    assert bool(s.isnan().all()) and not bool(q.float().any())
    # a row of zeros without eps is 0 * infinity
    assert bool(ks.rmsnorm_quantize(x[1:2], w, None, 0.0, dtype)[1].isnan().all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TOP)
@pytest.mark.parametrize("i", (1, 7, 8, 100, 256, 768, 1024, 1032, 2048, 2049, 8192, 28672, 32768))
def test_swiglu(i, dtype, kind):
    kind = KINDS[kind]
    for t in (1, 5, 331):
        if t * i > 4_000_000:
            continue
        x = rows(t, 2 * i, kind, i, 2.0)
        q, s = ks.swiglu_quantize(x, dtype)
        g, u = x[:, :i].double(), x[:, i:].double()
        check_codes(q, s, g * torch.sigmoid(g) * u, dtype)


def test_swiglu_extremes_and_strides():
    i = 64
    x = torch.zeros(6, 2 * i + 3, dtype=torch.float32, device="cuda")[:, :2 * i]
    x[0, 0], x[0, i] = -200.0, 3.0                           # exp(200) is infinite: the product is 0
    x[1, 1], x[1, i + 1] = 100.0, 2.0
    x[2, 0], x[2, i] = 1e20, 1e20                            # beyond fp32
    x[3, 5] = float("nan")
    x[4, 6], x[4, i + 6] = float("inf"), 1.0
    q, s = ks.swiglu_quantize(x)
    assert float(s[0]) == 0 and float(s[5]) == 0
    assert abs(float(s[1]) - 200.0 / 127) < 1e-6 and int(q[1, 1]) == 127
    for bad in (2, 3, 4):
        assert bool(s[bad].isnan()) and not bool(q[bad].any())


def test_empty_and_captured():
    w = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    q, s, _, _ = ks.rmsnorm_quantize(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16), w)
    assert q.shape == (0, 256) and s.shape == (0,)
    assert ks.swiglu_quantize(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16))[0].shape == (0, 128)
    x, r = rows(9, 256, torch.bfloat16, 1), rows(9, 256, torch.bfloat16, 2)
    want = [t.clone() for t in ks.rmsnorm_quantize(x, w, r)[:3]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ks.rmsnorm_quantize(x, w, r)
        again = ks.swiglu_quantize(got[2])
    x2 = rows(9, 256, torch.bfloat16, 3)
    graph.replay()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    x.copy_(x2)
    graph.replay()
    for a, b in zip(got[:3], ks.rmsnorm_quantize(x2, w, r)[:3]):
        assert torch.equal(a, b)
    assert torch.equal(again[0], ks.swiglu_quantize(got[2])[0])


@pytest.mark.parametrize("h", (24575, 24576, 24577, 31999))
def test_norm_of_wide_fp32_rows_off_vectors(h):
    """Rows whose two outputs share a place in shared memory, and the widest that have two; every output beside guard columns."""
    x, r, w = rows(3, h, torch.float32, 1, pad=3), rows(3, h, torch.float32, 2, pad=3), 1 + 0.1 * rows(1, h, torch.float32, 3)[0]
    he, y = norm_exact(x, w, r, 1e-6)
    wide = [torch.full((3, h + 3), -17, dtype=d, device="cuda") for d in (torch.int8, torch.float32, torch.float32)]
    q, s, hidden, n = ks.rmsnorm_quantize(x, w, r, out=(wide[0][:, 1:h + 1], None, wide[1][:, 2:h + 2], wide[2][:, 3:]))
    check_codes(q, s, y, torch.int8)
    assert torch.equal(hidden, x + r)
    assert bool(((n.double() - y).abs() <= 2 * REL * y.abs() + 1e-38).all())
    for b, first in zip(wide, (1, 2, 3)):
        assert bool((b[:, :first] == -17).all()) and bool((b[:, first + h:] == -17).all())


@pytest.mark.parametrize("kind", ("bf16", "fp32"))
@pytest.mark.parametrize("i", (64, 1025, 2048))
def test_swiglu_of_gates_far_below_zero(i, kind):
    """exp(-gate) leaves fp32 from -88.7 on while `up` may lift the product far above 2^-116: down to a gate of -170 nothing is lost.
    Tolerance in steps of 2^-23: an exponential of gate / 2 is off by two, and by what the roundings of its argument and of log2(e) move it, |gate| / 2 at most;
    it counts twice (its square); the reciprocal, the products and the scale add five: 9 + |gate|, and a tenth of that for their products."""
    pairs = [(-88.0, 1e10), (-87.5, 3e38), (-88.5, -1e5), (-100.0, 3e38), (-126.0, -1e38), (-140.0, 1e38), (-170.0, 3e38), (-60.0, 1e-3), (-1.0, 1e30), (-0.5, -2.0)]
    x = torch.zeros(len(pairs) + 2, 2 * i, device="cuda")
    for r, (g, u) in enumerate(pairs):
        x[r, 5], x[r, i + 5] = g, u
        x[r, 9], x[r, i + 9] = g, u / 2
    x[-2, 3], x[-2, i + 3] = -190.0, 3e38                    # 3e-42: below 2^-116
    x[-1, 3], x[-1, i + 3] = -3e38, 3e38
    x = x.to(KINDS[kind])
    g, u = x[:, :i].double(), x[:, i:].double()
    y = g * torch.sigmoid(g) * u
    for dtype, top in TOP.items():
        q, s = ks.swiglu_quantize(x, dtype)
        for r in range(len(pairs)):
            exact, steps = float(y[r].abs().max()) / top, (9 + float(g[r].abs().max())) * 1.1
            assert abs(float(s[r]) - exact) <= exact * steps * 2.0 ** -23, (r, float(s[r]), exact)
            sign = float(y[r, 5].sign())
            assert float(q[r, 5].float()) == sign * top and float(q[r, 9].float()) * sign in (64.0, 63.0, 224.0)
            assert int((q[r].float() != 0).sum()) == 2
        assert not bool(s[-2:].any()) and not bool(q[-2:].float().any())
