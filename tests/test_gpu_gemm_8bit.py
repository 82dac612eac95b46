"""The 8-bit products, dense and over experts' segments, against sums in 64 bits."""
import pytest
import torch

import kernelschema_b200 as ks

pytestmark = pytest.mark.gpu

CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
OUT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def codes(shape, kind, seed):
    """Codes over the whole range: int8 with -128 among them, e4m3 with its subnormals and largest values."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "int8":
        return torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8)
    x = torch.randn(shape, generator=g, device="cuda") * torch.exp2(torch.randint(-8, 7, shape, generator=g, device="cuda").float())
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def scales(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(n, generator=g, device="cuda") * 0.01 + 0.001


def check(out, a, sa, b, sb):
    """Each output within the roundings of the sum (none for int8; for e4m3 the 32 products and the partial sum of an instruction meet in fp32, so
    at most 33 of them lose half a step... taken as a whole step of the largest, which sum |a b| bounds), of the fp32 value of the sum, of two
    products with scales, and of the output's type."""
    f = sa.double()[:, None] * sb.double()[None, :]
    exact = (a.double() @ b.double().t()) * f
    tol = exact.abs() * (4 * 2.0 ** -24 + torch.finfo(out.dtype).eps / 2 * (1 + 2.0 ** -20))
    if a.dtype != torch.int8:
        tol += (a.double().abs() @ b.double().abs().t()) * f * (a.shape[1] + 32) * 1.1 * 2.0 ** -24
    if out.dtype == torch.float16:
        big = exact.abs() >= 65504                                # rounds to infinity from 65520 on
        assert bool((out[big].isinf() | (out[big].abs() == 65504)).all())
        exact, tol, out = exact[~big], tol[~big] + 2.0 ** -25, out[~big]   # half a step of the subnormals
    off = (out.double() - exact).abs()
    assert bool((off <= tol).all()), float((off - tol).max())


SHAPES = [(1, 128, 128), (1, 1, 16), (2, 129, 48), (15, 31, 112), (16, 127, 128), (17, 256, 144), (32, 100, 1024), (33, 384, 272), (64, 128, 4096),
          (65, 640, 512), (100, 2113, 528), (128, 96, 1040), (129, 128, 2048), (200, 1000, 640), (255, 130, 256), (256, 512, 400), (257, 77, 1536),
          (300, 4096, 256), (512, 1024, 1024), (1000, 333, 2064), (2049, 256, 768), (3, 4096, 7168), (8, 2048, 16384), (24, 7168, 2048), (1, 20000, 64)]
# one at least for each form that the library chooses among: few and many tiles of 16, 64 and 128 tokens, K split over 4 and 8 blocks, CTA pairs
SHAPES += [(1, 18470, 128), (9, 23005, 96), (16, 50, 14016), (5, 1223, 10112), (2, 4480, 3568), (17, 19156, 16), (22, 17, 1552), (627, 1, 2304), (17, 5243, 2896),
           (655, 1, 16), (666, 3164, 16), (651, 130, 1776), (1233, 20, 1968), (1339, 260, 5632), (1642, 1, 4288), (1642, 300, 4288), (897, 2509, 1344),
           (2500, 2700, 1040), (19053, 1, 16), (4097, 600, 2064), (16, 1, 25328), (3, 3070, 6800), (2, 4746, 3488), (25, 4244, 2992), (609, 1, 2528),
           (13, 1, 272), (9, 19119, 16), (32, 700, 1488), (12, 40, 192), (5, 33, 64)]


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_dense(m, n, k, kind):
    a, b, sa, sb = codes((m, k), kind, m), codes((n, k), kind, n + 1), scales(m, 3), scales(n, 4)
    for out_dtype in OUT.values():
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = ks.mm_8bit(a, sa, b, sb, out_dtype=out_dtype, status=status)
        assert out.dtype == out_dtype and out.shape == (m, n)
        check(out, a, sa, b, sb)
        assert int(status) == 0


@pytest.mark.parametrize("m", (1, 16, 100, 300))
def test_int8_sums_are_exact(m):
    """Products of like sign at the ends of the range, past 2^24, to the last bit; unit scales."""
    k = 16384
    a, b = torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.full((200, k), -128, dtype=torch.int8, device="cuda")
    b[1], b[2, ::2] = 127, 127
    a[0, 5] = 3
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(200, device="cuda")
    out = ks.mm_8bit(a, one_m, b, one_n, out_dtype=torch.float32)
    assert torch.equal(out, (a.double() @ b.double().t()).float())


def test_int8_longest_k():
    k = 131056
    a, b = codes((3, k), "int8", 1), codes((5, k), "int8", 2)
    a[0], b[0] = -128, -128
    out = ks.mm_8bit(a, torch.ones(3, device="cuda"), b, torch.ones(5, device="cuda"), out_dtype=torch.float32)
    assert torch.equal(out, (a.double() @ b.double().t()).float())


@pytest.mark.parametrize("m", (1, 20, 70, 300))
def test_strides_and_guards(m):
    """Rows of a and out inside wider buffers; a scale column; nothing beside the output is written."""
    k, n = 256, 131
    wide = codes((m, k + 48), "int8", 1)
    a, b, sa, sb = wide[:, 16:16 + k], codes((n, k), "int8", 2), scales(m, 3), scales(n, 4)
    back = torch.full((m + 2, n + 5), -17.0, dtype=torch.bfloat16, device="cuda")
    out = ks.mm_8bit(a, sa[:, None], b, sb[:, None], out=back[1:-1, 3:-2])
    assert out.data_ptr() == back[1:-1, 3:-2].data_ptr()
    check(out, a, sa, b, sb)
    back[1:-1, 3:-2] = -17.0
    assert bool((back == -17).all())
    check(ks.mm_8bit(wide[:, 3:3 + k], sa, b, sb), wide[:, 3:3 + k], sa, b, sb)      # off 16 bytes: read as a copy
    tall = torch.empty(k, m, dtype=torch.int8, device="cuda").copy_(a.t()).t()       # columns first
    check(ks.mm_8bit(tall, sa, b, sb), a, sa, b, sb)


def test_special_values():
    """A NaN scale (a row without a finite peak) makes its row NaN and no other; a zero scale makes zeros; e4m3 NaN codes stay in their row."""
    for kind in CODES:
        a, b, sa, sb = codes((40, 128), kind, 1), codes((140, 128), kind, 2), scales(40, 3), scales(140, 4)
        sa[3], sa[4] = float("nan"), 0.0
        if kind == "e4m3":
            a.view(torch.uint8)[7, 9] = 0x7F
        out = ks.mm_8bit(a, sa, b, sb)
        assert bool(out[3].isnan().all()) and not bool(out[4].any())
        rows = [r for r in range(40) if r not in (3, 4, 7)] + ([7] if kind == "int8" else [])
        check(out[rows], a[rows], sa[rows], b, sb)
        assert kind == "int8" or bool(out[7].isnan().all())


def segments(counts, lead=0):
    off = [lead]
    for c in counts:
        off.append(off[-1] + c)
    return torch.tensor(off, dtype=torch.int32, device="cuda")


GROUPS = [([1], 0), ([0, 0, 5, 0], 0), ([3, 0, 17, 1, 64, 65, 0, 2], 0), ([16] * 40, 5), ([100, 130, 0, 257, 1, 300, 511, 33], 0), ([1] * 200, 56),
          ([0] * 7, 9), ([1000], 0), ([128, 256, 384], 1), ([7] * 33 + [0] * 31, 0)]


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("n,k", ((128, 128), (200, 272), (33, 1040)))
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_grouped(case, n, k, kind):
    counts, behind = GROUPS[case]
    e, m = len(counts), sum(counts) + behind
    off = segments(counts)
    a, b, sa, sb = codes((m, k), kind, 1), codes((e, n, k), kind, 2), scales(m, 3), scales(e * n, 4).view(e, n)
    for out_dtype in (torch.bfloat16, torch.float32):
        out = ks.mm_8bit_grouped(a, sa, b, sb, off, out_dtype=out_dtype)
        given = torch.full((m, n + 3), -17.0, dtype=out_dtype, device="cuda")
        ks.mm_8bit_grouped(a, sa, b, sb, off, out=given[:, 1:-2])
        assert torch.equal(given[:sum(counts), 1:-2], out[:sum(counts)])
        assert bool((given[sum(counts):] == -17).all()) and bool((given[:, 0] == -17).all()) and bool((given[:, -2:] == -17).all())
        assert not bool(out[sum(counts):].any())
        at = off.tolist()
        for i in range(e):
            if counts[i]:
                check(out[at[i]:at[i + 1]], a[at[i]:at[i + 1]], sa[at[i]:at[i + 1]], b[i], sb[i])


def test_grouped_offsets_that_are_none():
    """A start above zero, and offsets that fall or leave the rows: cut to what there is."""
    a, b, sa, sb = codes((90, 64), "int8", 1), codes((3, 40, 64), "int8", 2), scales(90, 3), scales(120, 4).view(3, 40)
    out = ks.mm_8bit_grouped(a, sa, b, sb, segments([10, 0, 20], lead=30))
    assert not bool(out[:30].any()) and not bool(out[60:].any())
    check(out[30:40], a[30:40], sa[30:40], b[0], sb[0])
    check(out[40:60], a[40:60], sa[40:60], b[2], sb[2])
    odd = torch.tensor([-5, 50, 20, 1 << 30], dtype=torch.int32, device="cuda")      # 0..50, none, 50..90
    out = ks.mm_8bit_grouped(a, sa, b, sb, odd)
    check(out[:50], a[:50], sa[:50], b[0], sb[0])
    check(out[50:], a[50:], sa[50:], b[2], sb[2])


def test_grouped_many_experts():
    e, n, k = 1024, 16, 32
    counts = [(i * 7) % 5 for i in range(e)]
    a, b = codes((sum(counts), k), "int8", 1), codes((e, n, k), "int8", 2)
    sa, sb = scales(sum(counts), 3), scales(e * n, 4).view(e, n)
    out = ks.mm_8bit_grouped(a, sa, b, sb, segments(counts), out_dtype=torch.float32)
    which = torch.repeat_interleave(torch.arange(e, device="cuda"), torch.tensor(counts, device="cuda"))
    exact = torch.einsum("mk,mnk->mn", a.double(), b.double()[which]) * sa.double()[:, None] * sb.double()[which]
    assert bool(((out.double() - exact).abs() <= exact.abs() * 6 * 2.0 ** -24).all())


def test_empty_captured_and_repeated():
    b, sb = codes((140, 256), "int8", 2), scales(140, 4)
    assert ks.mm_8bit(codes((0, 256), "int8", 1), scales(0, 1), b, sb).shape == (0, 140)
    a, sa = codes((33, 256), "int8", 5), scales(33, 6)
    off = segments([11, 0, 20])
    b3, sb3 = codes((3, 140, 256), "int8", 7), scales(420, 8).view(3, 140)
    want = ks.mm_8bit(a, sa, b, sb), ks.mm_8bit_grouped(a, sa, b3, sb3, off)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ks.mm_8bit(a, sa, b, sb), ks.mm_8bit_grouped(a, sa, b3, sb3, off)
    for _ in range(3):
        graph.replay()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    a2 = codes((33, 256), "int8", 9)
    a.copy_(a2)
    off.copy_(segments([5, 6, 22]))
    graph.replay()
    check(got[0], a2, sa, b, sb)
    check(got[1][5:11], a2[5:11], sa[5:11], b3[1], sb3[1])
    # two streams at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append([ks.mm_8bit(a, sa, b, sb) for _ in range(20)])
    torch.cuda.synchronize()
    for o in outs[0] + outs[1]:
        assert torch.equal(o, got[0])


# the forms that the shapes above leave out for one type of codes or for both (which form a call takes: test_host_rules.py)
MORE_SHAPES = [(1, 4861, 5312), (3, 5425, 3376), (1, 2401, 12800), (5, 2959, 6960), (9, 1001, 24592), (16, 513, 32784), (17, 5513, 3568), (19, 4175, 2880), (391, 591, 4528),
               (683, 123, 1744), (677, 125, 3344)]


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("m,n,k", MORE_SHAPES)
def test_dense_of_the_other_forms(m, n, k, kind):
    test_dense(m, n, k, kind)


# (counts, rows behind, first row): on CTA pairs above 160 rows a segment, K >= 1536 and N > 128; single tiles of 64 and 128 that are more than the device runs at once
MORE_GROUPS = [([100, 700, 0, 257, 1, 513, 333, 161], 57, 3, 200, 1536), ([100, 700, 0, 257, 1, 513, 333, 161], 0, 0, 384, 2064), ([300, 150] * 10, 9, 65, 129, 1552),
               ([1500], 1, 2, 2049, 1536), ([0, 1025, 0, 32, 511, 224], 300, 1, 1000, 1600), ([20] * 30, 2, 1, 1000, 272), ([40] * 30, 5, 7, 1000, 272), ([200, 0, 64, 33] * 8, 3, 0, 384, 2064)]


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("case", range(len(MORE_GROUPS)))
def test_grouped_of_the_other_forms(case, kind):
    """Uneven segments that start anywhere, tiles of 32 to 256 rows, weight rows of the next expert in a tile, rows in front of and behind the segments."""
    counts, behind, lead, n, k = MORE_GROUPS[case]
    e, m, end = len(counts), lead + sum(counts) + behind, lead + sum(counts)
    off = segments(counts, lead)
    a, b, sa, sb = codes((m, k), kind, 1), codes((e, n, k), kind, 2), scales(m, 3), scales(e * n, 4).view(e, n)
    at = off.tolist()
    for out_dtype in (torch.bfloat16, torch.float32):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = ks.mm_8bit_grouped(a, sa, b, sb, off, out_dtype=out_dtype, status=status)
        given = torch.full((m, n + 3), -17.0, dtype=out_dtype, device="cuda")
        ks.mm_8bit_grouped(a, sa, b, sb, off, out=given[:, 1:-2], status=status)
        assert int(status) == 0
        assert torch.equal(given[lead:end, 1:-2], out[lead:end]) and not bool(out[:lead].any()) and not bool(out[end:].any())
        assert bool((given[:lead] == -17).all()) and bool((given[end:] == -17).all()) and bool((given[:, 0] == -17).all()) and bool((given[:, -2:] == -17).all())
        for i in range(e):
            if counts[i]:
                check(out[at[i]:at[i + 1]], a[at[i]:at[i + 1]], sa[at[i]:at[i + 1]], b[i], sb[i])


@pytest.mark.parametrize("kind", CODES)
@pytest.mark.parametrize("m,n,k", ((1, 200, 512), (5, 192, 512), (64, 192, 512), (700, 512, 192), (700, 384, 1536)))
def test_dense_and_grouped_agree(m, n, k, kind):
    """One segment of all rows is the dense product: the same bits in int8, sums in another order in e4m3."""
    a, b, sa, sb = codes((m, k), kind, 1), codes((n, k), kind, 2), scales(m, 3), scales(n, 4)
    dense, grouped = ks.mm_8bit(a, sa, b, sb), ks.mm_8bit_grouped(a, sa, b[None], sb[None], segments([m]))
    check(dense, a, sa, b, sb)
    check(grouped, a, sa, b, sb)
    assert kind == "e4m3" or torch.equal(dense, grouped)
