"""Arguments that the 8-bit operators refuse, checked before any device work (no GPU needed)."""
import pytest
import torch

import kernelschema_b200 as ks


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
