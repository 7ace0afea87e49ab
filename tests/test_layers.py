"""Refusals of the normalised-linear operators.  Every argument is checked
before the first CUDA call, so these run without a GPU."""

import ctypes

import pytest

from burn_automata_b200 import Activation, _lib
from burn_automata_b200 import config as C
from burn_automata_b200 import layers

BUF = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(BUF) + 255) // 256 * 256  # never dereferenced: refused first


def norm(lib, dtype=0, x=AT, xs=8, w=AT, b=AT, rows=2, dims=8, eps=1e-5, y=AT, ys=8, mean=AT,
         rstd=AT):
    return lib.npa_dev_layer_norm(dtype, x, xs, w, b, rows, dims, eps, y, ys, mean, rstd, None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), 8), (dict(dtype=-1), 8), (dict(rows=-1), 8), (dict(dims=0), 8),
    (dict(rows=1 << 31), 24), (dict(dims=(1 << 24) + 1, xs=1 << 25, ys=1 << 25), 24),
    (dict(x=None), 8), (dict(y=None), 8), (dict(xs=7), 8), (dict(ys=7), 8), (dict(xs=-8), 8),
    (dict(x=AT + 2), 8), (dict(mean=AT + 2), 8), (dict(dtype=1, x=AT + 1), 8),
    (dict(eps=0.0), 2), (dict(eps=-1e-5), 2), (dict(eps=float("nan")), 2),
    (dict(eps=float("inf")), 2), (dict(xs=1 << 41), 24),
])
def test_layer_norm_refuses(npa_lib, kw, status):
    assert norm(npa_lib, **kw) == status
    assert npa_lib.npa_last_error_message()


def test_layer_norm_without_rows_needs_no_buffers(npa_lib):
    assert norm(npa_lib, rows=0, x=None, y=None, mean=None, rstd=None) == 0


def norm_backward(lib, dtype=0, dy=AT, dys=8, x=AT, xs=8, mean=AT, rstd=AT, w=AT, res=None, rs=0,
                  rows=2, dims=8, dx=AT, dxs=8, dw=AT, db=AT, ws=AT, ws_bytes=1 << 30):
    return lib.npa_dev_layer_norm_backward(dtype, dy, dys, x, xs, mean, rstd, w, res, rs, rows,
                                           dims, dx, dxs, dw, db, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=9), 8), (dict(rows=-3), 8), (dict(dims=0), 8), (dict(dy=None), 8),
    (dict(x=None), 8), (dict(mean=None), 8), (dict(rstd=None), 8), (dict(dys=3), 8),
    (dict(dxs=3), 8), (dict(res=AT, rs=3), 8), (dict(res=AT, rs=8, dx=None), 8),
    (dict(ws=None), 8), (dict(ws_bytes=8), 8), (dict(ws=AT + 4), 8),
])
def test_layer_norm_backward_refuses(npa_lib, kw, status):
    assert norm_backward(npa_lib, **kw) == status


def linear(lib, dtype=0, act=0, x=AT, xs=8, w=AT, ws_=8, b=AT, r=None, rs=0, rows=2, inputs=8,
           outputs=4, y=AT, ys=4, z=None, zs=0, work=AT, work_bytes=1 << 30):
    return lib.npa_dev_linear(dtype, act, x, xs, w, ws_, b, r, rs, rows, inputs, outputs, y, ys, z,
                              zs, work, work_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=7), 8), (dict(act=5), 8), (dict(act=-1), 8), (dict(rows=-1), 8),
    (dict(inputs=0), 8), (dict(outputs=0), 8), (dict(inputs=1 << 25, xs=1 << 25, ws_=1 << 25), 24),
    (dict(x=None), 8), (dict(w=None), 8), (dict(y=None), 8), (dict(xs=7), 8), (dict(ws_=7), 8),
    (dict(ys=3), 8), (dict(r=AT, rs=3), 8), (dict(z=AT, zs=3), 8), (dict(y=AT + 1), 8),
])
def test_linear_refuses(npa_lib, kw, status):
    assert linear(npa_lib, **kw) == status


def linear_backward(lib, dtype=0, act=1, dy=AT, dys=4, x=AT, xs=8, w=AT, ws_=8, z=AT, zs=4, rows=2,
                    inputs=8, outputs=4, dx=AT, dxs=8, dw=AT, db=AT, work=AT, work_bytes=1 << 30):
    return lib.npa_dev_linear_backward(dtype, act, dy, dys, x, xs, w, ws_, z, zs, rows, inputs,
                                       outputs, dx, dxs, dw, db, work, work_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=7), 8), (dict(act=5), 8), (dict(rows=-1), 8), (dict(inputs=0), 8),
    (dict(outputs=0), 8), (dict(dy=None), 8), (dict(x=None), 8), (dict(w=None), 8),
    (dict(z=None), 8), (dict(dys=3), 8), (dict(zs=3), 8), (dict(dxs=7), 8), (dict(ws_=7), 8),
    (dict(work=None), 8), (dict(work_bytes=1), 8), (dict(work=AT + 16), 8),
])
def test_linear_backward_refuses(npa_lib, kw, status):
    assert linear_backward(npa_lib, **kw) == status


def test_workspace_queries_refuse_and_answer(npa_lib):
    n = ctypes.c_size_t(0)
    q = npa_lib.npa_dev_layer_norm_backward_workspace_size
    assert q(0, 100, 64, ctypes.byref(n)) == 0 and n.value > 0
    assert q(0, 100, 0, ctypes.byref(n)) == 8
    assert q(0, 100, 64, None) == 8
    q = npa_lib.npa_dev_linear_backward_workspace_size
    assert q(2, 1, 100, 64, 32, ctypes.byref(n)) == 0 and n.value > 0
    assert q(2, 9, 100, 64, 32, ctypes.byref(n)) == 8
    q = npa_lib.npa_dev_linear_workspace_size
    assert q(2, 100, 64, 32, ctypes.byref(n)) == 0
    assert q(2, -1, 64, 32, ctypes.byref(n)) == 8


def test_python_layer_refuses_what_it_cannot_take():
    torch = pytest.importorskip("torch")
    x = torch.zeros(2, 8)
    for call in (lambda: layers.layer_norm(x), lambda: layers.layer_norm([1.0]),
                 lambda: layers.linear(x, torch.zeros(4, 8)),
                 lambda: layers.layer_norm(x.double()), lambda: layers.layer_norm(x.long())):
        with pytest.raises(C.InvalidArgument):
            call()
    assert Activation.Silu == 4
    assert _lib.lib().npa_abi_version() == 1


def test_operands_off_16_bytes_are_copied_where_it_pays():
    """By the stride and by the address alike; small products, f32 operands that
    few outputs read and rows that a copy would not align stay in place."""
    torch = pytest.importorskip("torch")
    big = 1 << 30

    def at(rows, width, offset, pitch, dtype):
        # a start on 16 bytes, whatever the allocator gives
        flat = torch.zeros(rows * (width + pitch) + offset + 16, dtype=dtype)
        start = -flat.data_ptr() % 16 // flat.element_size() + offset
        return flat[start:start + rows * (width + pitch)].view(rows, width + pitch)[:, :width]

    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        for offset, pitch, copied in ((0, 0, False), (1, 0, True), (0, 1, True), (3, 8, True),
                                      (0, 8, False), (8, 0, False)):
            t = at(64, 32, offset, pitch, dtype)
            t += torch.arange(64 * 32).view(64, 32).to(dtype) / 64
            got, stride = layers._aligned_rows(t, big, 1024)
            assert (got.data_ptr() != t.data_ptr()) == copied, (dtype, offset, pitch)
            assert torch.equal(got, t) and stride == (32 if copied else 32 + pitch)
            if copied:
                assert got.data_ptr() % 16 == 0 and got.is_contiguous()
            assert layers._aligned_rows(t, big - 1, 1024)[0].data_ptr() == t.data_ptr()
            few = layers._aligned_rows(t, big, 128)[0]
            assert (few.data_ptr() != t.data_ptr()) == (copied and dtype != torch.float32)
    odd = at(64, 33, 1, 0, torch.bfloat16)
    assert layers._aligned_rows(odd, big, 1024)[0].data_ptr() == odd.data_ptr()
