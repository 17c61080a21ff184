"""The workspace of the C entries of the linear layers: what they refuse before they reach a device, and the least
alignment that they take."""
import ctypes as C

import pytest

from splatx_cuda import _native as n

AT = 1 << 20  # an address that nothing reads: every call here is refused


@pytest.fixture
def lib():
    if not n.library_path().exists():
        pytest.skip("library not built")
    return n.lib()


@pytest.mark.parametrize("dtype, align", [(0, 16), (1, 32), (2, 32)])
def test_linear_workspace_alignment(lib, dtype, align):
    """Parts of 16-bit tiles that are cut along K leave 32 bytes at a time. x and weight start on an odd element: the
    16-bit calls need a copy of each, so that one byte is too small whatever else is asked."""
    size = 4 if dtype == 0 else 2
    ins = n.SxLinearInputs(AT + size, AT + size, None, 300, 4096, 256, 4096, 4096, dtype, 0, 0)
    out = n.SxLinearOutputs(None, 0, AT, 256, None, 0)
    gin, gout = n.SxLinearGradsIn(AT, 256, None, 0), n.SxLinearGrads(AT, 4096, AT, 4096, AT)
    for off in {align // 2, 8, 4, 1}:
        for call in (lambda ws, b: lib.sxcuda_linear_fwd(C.byref(ins), C.byref(out), ws, C.byref(b), None),
                     lambda ws, b: lib.sxcuda_linear_bwd(C.byref(ins), C.byref(gin), C.byref(gout), ws, C.byref(b), None)):
            assert call(AT + off, C.c_size_t(1)) == n.SXCUDA_EINVAL
            assert f"{align}-byte aligned" in lib.sxcuda_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, align", [("float32", 16), ("float16", 32), ("bfloat16", 32)])
def test_linear_least_alignment(lib, dtype, align):
    """Products that are cut along K, on a workspace that starts on no more than it has to."""
    import torch
    from splatx_cuda import network
    T, code = getattr(torch, dtype), {"float32": 0, "float16": 1, "bfloat16": 2}[dtype]
    gen = torch.Generator().manual_seed(1)

    def run(entry, *args):
        nbytes, args = C.c_size_t(0), [C.byref(a) for a in args]
        n.check(entry(*args, None, C.byref(nbytes), None))
        assert nbytes.value > 0
        ws = torch.empty(nbytes.value + align, dtype=torch.uint8, device="cuda")
        assert ws.data_ptr() % 64 == 0
        n.check(entry(*args, ws.data_ptr() + align, C.byref(nbytes), torch.cuda.current_stream().cuda_stream))

    for m, k, o in ((300, 4096, 256), (8000, 4096, 264)):  # the forward is cut, the weight's gradient is
        x, w, g = (torch.randn(s, generator=gen).to(T).cuda() for s in ((m, k), (o, k), (m, o)))
        y, v_x, v_w = torch.empty_like(g), torch.empty_like(x), torch.empty_like(w)
        ins = n.SxLinearInputs(x.data_ptr(), w.data_ptr(), None, m, k, o, k, k, code, 0, 0)
        if m == 300:
            run(lib.sxcuda_linear_fwd, ins, n.SxLinearOutputs(None, 0, y.data_ptr(), o, None, 0))
            assert torch.equal(y, network.linear_fwd(x, w)[0])
        else:
            run(lib.sxcuda_linear_bwd, ins, n.SxLinearGradsIn(g.data_ptr(), o, None, 0), n.SxLinearGrads(v_x.data_ptr(), k, v_w.data_ptr(), k, None))
            assert all(torch.equal(a, b) for a, b in zip((v_x, v_w), network.linear_bwd(g, x, w)))
