"""Arguments that the 8-bit operators refuse, checked before any device work (no GPU needed)."""
import os
import re

import pytest
import torch

import kernelschema_b200 as ks

CSRC = os.path.join(os.path.dirname(os.path.abspath(ks.__file__)), "csrc")


@pytest.fixture(scope="module")
def lib():
    from kernelschema_b200 import _lib, build
    build.build()
    return _lib.load()


def z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def test_rowquant_refusals():
    for call in (lambda: ks.rmsnorm_quantize(z(4, 64), z(64)),                                       # not on a device
                 lambda: ks.swiglu_quantize(z(4, 64)),
                 lambda: ks.rmsnorm_quantize(z(4, 64, dtype=torch.int8), z(64, dtype=torch.int8)),
                 lambda: ks.rmsnorm_quantize(z(4, 4, 64), z(64)),
                 lambda: ks.rmsnorm_quantize(z(4, 64), z(63)),
                 lambda: ks.rmsnorm_quantize(z(4, 64), z(64, dtype=torch.float16)),
                 lambda: ks.rmsnorm_quantize(z(4, 64), z(64), z(3, 64)),
                 lambda: ks.rmsnorm_quantize(z(4, 64), z(64), z(4, 64, dtype=torch.float32)),
                 lambda: ks.rmsnorm_quantize(z(4, 64), z(64), dtype=torch.uint8),
                 lambda: ks.swiglu_quantize(z(4, 63)),
                 lambda: ks.swiglu_quantize(z(4, 64), dtype=torch.float8_e5m2)):
        with pytest.raises(ValueError):
            call()


def test_rowquant_abi_refusals(lib):
    def norm(x=16, xs=64, r=None, rs=0, w=16, wt=0, rows=4, cols=64, eps=1e-6, dt=0, qt=0, q=16, qs=64, sc=16, hid=None, hs=0, n=None, ns=0):
        return lib.b200moe_rmsnorm_quantize(x, xs, r, rs, w, wt, rows, cols, eps, dt, qt, q, qs, sc, hid, hs, n, ns, None)

    assert norm(cols=0) == 775 and norm(cols=32769) == 775 and norm(rows=-1) == 775 and norm(rows=1 << 31) == 775
    assert norm(dt=3) == 776 and norm(qt=2) == 776 and norm(wt=1) == 776 and norm(eps=-1.0) == 776 and norm(eps=float("nan")) == 776
    assert norm(x=None) == 777 and norm(w=None) == 777 and norm(q=None) == 777 and norm(sc=None) == 777
    assert norm(x=17) == 778 and norm(qs=63) == 778 and norm(hid=16, hs=63) == 778 and norm(n=18, ns=64, dt=2, wt=2) == 778 and norm(sc=18) == 778
    assert norm(xs=-64) == 778 and norm(r=16, rs=-1) == 778
    assert norm(rows=0, x=None) == 0

    def swi(x=16, xs=128, rows=4, cols=64, dt=0, qt=0, q=16, qs=64, sc=16):
        return lib.b200moe_swiglu_quantize(x, xs, rows, cols, dt, qt, q, qs, sc, None)

    assert swi(cols=0) == 779 and swi(cols=32769) == 779 and swi(dt=-1) == 776 and swi(qt=5) == 776 and swi(x=None) == 777
    assert swi(x=18, dt=2) == 778 and swi(qs=1) == 778 and swi(xs=-1) == 778 and swi(rows=0, q=None) == 0
    assert b"swiglu_quantize" in lib.b200moe_last_error()


def test_gemm_8bit_refusals(lib):
    i8 = torch.int8
    f = torch.float32
    ok = dict(a=z(4, 64, dtype=i8), sa=z(4, dtype=f), b=z(32, 64, dtype=i8), sb=z(32, dtype=f))

    def mm(out=None, out_dtype=torch.bfloat16, status=None, **over):
        v = dict(ok, **over)
        return ks.mm_8bit(v["a"], v["sa"], v["b"], v["sb"], out, out_dtype, status)

    for over in (dict(),                                                                              # not on a device
                 dict(a=z(4, 64)), dict(b=z(32, 64, dtype=torch.float8_e4m3fn)), dict(b=z(32, 48, dtype=i8)), dict(a=z(4, 60, dtype=i8), b=z(32, 60, dtype=i8)),
                 dict(sa=z(5, dtype=f)), dict(sb=z(31, dtype=f)), dict(sa=z(4)), dict(out_dtype=torch.int32), dict(a=z(2, 4, 64, dtype=i8)),
                 dict(status=z(1, dtype=f)), dict(a=z(4, 0, dtype=i8), b=z(32, 0, dtype=i8)), dict(b=z(0, 64, dtype=i8), sb=z(0, dtype=f))):
        with pytest.raises(ValueError):
            mm(**over)
    b3, s3, off = z(3, 32, 64, dtype=i8), z(3, 32, dtype=f), z(4, dtype=torch.int32)
    for args in ((ok["a"], ok["sa"], b3, s3, off), (ok["a"], ok["sa"], b3, s3, z(3, dtype=torch.int32)), (ok["a"], ok["sa"], b3, s3, z(4, dtype=torch.int64)),
                 (ok["a"], ok["sa"], ok["b"], ok["sb"], off), (ok["a"], ok["sa"], b3, ok["sb"], off)):
        with pytest.raises(ValueError):
            ks.mm_8bit_grouped(*args)

    def abi(a=16, a_st=64, sa=16, b=16, sb=16, out=16, m=4, n=32, k=64, o_st=32, code=0, ot=0, off=None, e=None):
        if e is None:
            return lib.b200moe_gemm_8bit(a, a_st, sa, b, sb, out, m, n, k, o_st, code, ot, None, None)
        return lib.b200moe_gemm_8bit_grouped(a, a_st, sa, b, sb, off, e, out, m, n, k, o_st, code, ot, 0, None, None)

    assert abi(k=60) == 784 and abi(k=131072) == 784 and abi(n=0) == 784 and abi(m=-1) == 784 and abi(m=(1 << 30) + 1) == 784
    assert abi(code=2) == 785 and abi(ot=3) == 785 and abi(a=None) == 786 and abi(sb=None) == 786 and abi(out=None) == 786
    assert abi(a=24) == 783 and abi(b=8) == 783 and abi(a_st=48) == 783 and abi(a_st=72) == 783 and abi(o_st=31) == 783 and abi(out=17) == 783
    assert abi(m=0, a=None) == 0 and abi(e=0, off=16) == 784 and abi(e=1025, off=16) == 784 and abi(e=3) == 786 and abi(e=3, off=18) == 783
    assert abi(e=1024, off=16, n=1 << 21) == 784


def test_route_order_refusals(lib):
    i32 = torch.int32
    ids = z(4, 2, dtype=i32)
    order = ks.RouteOrder(z(9, dtype=i32), ids, z(8, dtype=i32))
    for call in (lambda: ks.route_sort(ids, 8),                                                       # not on a device
                 lambda: ks.route_sort(ids.long(), 8), lambda: ks.route_sort(ids[0], 8), lambda: ks.route_sort(ids, 0), lambda: ks.route_sort(ids, 1025),
                 lambda: ks.route_sort(z(4, 0, dtype=i32), 8),
                 lambda: ks.sort_tokens(z(4, 64), order), lambda: ks.sort_tokens(z(5, 64), order), lambda: ks.sort_tokens(z(4, 64, dtype=torch.float64), order),
                 lambda: ks.sort_tokens(z(4, 2, 2), order), lambda: ks.sort_tokens(z(4, 0), order),
                 lambda: ks.sort_tokens(z(4, 64), order._replace(row_of=ids.long())), lambda: ks.sort_tokens(z(4, 64), order._replace(row_of=ids.t())),
                 lambda: ks.unsort_tokens(z(8, 64), order), lambda: ks.unsort_tokens(z(4, 64), order), lambda: ks.unsort_tokens(z(8, 64, dtype=torch.int8), order),
                 lambda: ks.unsort_tokens(z(8, 64), order, z(4, 2)), lambda: ks.unsort_tokens(z(8, 64), order, z(2, 4, dtype=torch.float32))):
        with pytest.raises(ValueError):
            call()

    size = lib.b200moe_route_sort_workspace_bytes
    assert size(1024, 8, 128) == 0 and size(1025, 8, 128) == 10 * 129 * 4 and size(1, 1, 1025) == -1 and size(1 << 28, 8, 4) == -1 and size(-1, 8, 4) == -1

    def sort(ids=16, st=8, t=4, k=8, e=16, off=16, row=16, inv=16, ws=None, wb=0):
        return lib.b200moe_route_sort(ids, st, t, k, e, off, row, inv, ws, wb, None)

    assert sort(t=-1) == 787 and sort(k=0) == 787 and sort(t=1 << 28) == 787 and sort(e=0) == 787 and sort(e=1025) == 787
    assert sort(ids=None) == 788 and sort(off=None) == 788 and sort(inv=None) == 788 and sort(st=-1) == 789 and sort(row=18) == 789
    assert sort(t=4096) == 771 and sort(t=4096, ws=16, wb=100) == 771

    def rows(x=16, st=64, t=4, rb=64, row=16, k=2, valid=16, out=16):
        return lib.b200moe_sort_rows(x, st, t, rb, row, k, valid, out, None)

    assert rows(t=1 << 26) == 787 and rows(rb=0) == 787 and rows(t=-1) == 787 and rows(k=0) == 787 and rows(x=None) == 788 and rows(valid=None) == 788 and rows(st=-1) == 789
    assert rows(row=18) == 789 and rows(t=0, x=None) == 0

    def back(r=16, rs=64, n=8, row=16, w=None, t=4, k=2, c=64, dt=0, out=16, os=64):
        return lib.b200moe_unsort_rows(r, rs, n, row, w, t, k, c, dt, out, os, None)

    assert back(t=1 << 26) == 787 and back(c=0) == 787 and back(dt=3) == 787 and back(n=-1) == 787 and back(r=None) == 788 and back(row=None) == 788 and back(os=63) == 788
    assert back(rs=-1) == 789 and back(r=17) == 789 and back(w=18) == 789 and back(t=0, r=None) == 0

    def grad(g=16, gs=64, r=16, rs=64, row=16, w=16, t=4, k=2, c=64, dt=0, valid=16, gr=16, gw=16):
        return lib.b200moe_unsort_rows_backward(g, gs, r, rs, row, w, t, k, c, dt, valid, gr, gw, None)

    assert grad(c=0) == 787 and grad(g=None) == 788 and grad(valid=None) == 788 and grad(r=None) == 788 and grad(gr=17) == 789 and grad(gw=18) == 789
    assert grad(gr=None, gw=None) == 0 and grad(t=0) == 0


def test_tangents_are_refused():
    """Forward-mode differentiation would lose its tangent (a dual tensor does not require a gradient), so the sorting calls refuse it."""
    import torch.autograd.forward_ad as forward_ad
    i32, f = torch.int32, torch.float32
    order = ks.RouteOrder(z(9, dtype=i32), z(4, 2, dtype=i32), z(8, dtype=i32))
    with forward_ad.dual_level():
        dual = lambda v: forward_ad.make_dual(v, torch.ones_like(v))  # noqa: E731
        for call in (lambda: ks.sort_tokens(dual(z(4, 64)), order), lambda: ks.sort_tokens(dual(z(4, dtype=f)), order), lambda: ks.unsort_tokens(dual(z(8, 64)), order),
                     lambda: ks.unsort_tokens(z(8, 64), order, dual(z(4, 2, dtype=f))), lambda: ks.unsort_tokens(z(8, 64).requires_grad_(), order, dual(z(4, 2, dtype=f)))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):     # which leaves forward mode on
                call()
        x = dual(z(4, 64))
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA"):
            ks.sort_tokens(x, order)                               # no tangent is asked for: a call like any other


def test_8bit_operators_refuse_tensors_that_want_a_derivative():
    """The results of the 8-bit operators hang on no graph: an input that requires a gradient, or has a tangent, is refused instead of losing it."""
    import torch.autograd.forward_ad as forward_ad
    i8, f, e4m3 = torch.int8, torch.float32, torch.float8_e4m3fn
    off = z(2, dtype=torch.int32)
    grouped = lambda a, sa, b, sb, out=None: ks.mm_8bit_grouped(a, sa, b[None], sb[None], off, out)  # noqa: E731
    norm = lambda x, w, r, hidden, normed: ks.rmsnorm_quantize(x, w, r, out=(None, None, hidden, normed))  # noqa: E731
    swiglu = lambda x, s: ks.swiglu_quantize(x, out=(None, s))  # noqa: E731
    x, w, codes = z(4, 64), z(64), (z(4, 64, dtype=i8), z(32, 64, dtype=i8))
    for call, args, named in ((norm, (x, w, x, x, x), "rmsnorm_quantize"), (swiglu, (x, z(4, dtype=f)), "swiglu_quantize"),
                              (ks.mm_8bit, (codes[0], z(4, dtype=f), codes[1], z(32, dtype=f), z(4, 32)), "mm_8bit"),
                              (grouped, (codes[0], z(4, dtype=f), codes[1], z(32, dtype=f), z(4, 32)), "mm_8bit_grouped"),
                              (ks.mm_8bit, (z(4, 64, dtype=e4m3), z(4, dtype=f), z(32, 64, dtype=e4m3), z(32, dtype=f)), "mm_8bit")):
        for i, v in enumerate(args):
            if not v.is_floating_point():
                continue
            wants = args[:i] + (v.clone().requires_grad_(),) + args[i + 1:]
            with pytest.raises(ValueError, match=named + " has no gradient"):
                call(*wants)
            with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):         # nothing is asked for: a call like any other
                call(*wants)
            if v.dtype == e4m3:
                continue
            with forward_ad.dual_level(), pytest.raises(ValueError, match=named + " has no forward-mode"):
                call(*args[:i], forward_ad.make_dual(v, torch.ones_like(v)), *args[i + 1:])


def test_cluster_kernels_in_headers_let_nothing_in_early():
    """The rule for cluster kernels holds for those in headers: released by their end alone, they have no pdl_trigger."""
    seen = set()
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith(".cuh"):
            continue
        text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        for kernel in re.split(r"\b__global__\b", text)[1:]:
            body = kernel[:kernel.index("\n}\n")]
            if "cluster" in body:
                seen.add(re.search(r"\b(k_\w+)\s*\(", body).group(1))
                assert "pdl_trigger" not in body, name
    assert seen == {"k_gemm_8bit_pair", "k_gemm_8bit_split"}
