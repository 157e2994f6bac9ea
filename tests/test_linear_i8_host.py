"""The 8-bit linear path without a GPU: what its entry points refuse on the host, and the row layout."""
import ctypes
import os
import re

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from streaming_sparse_b200 import ops


@pytest.fixture(scope="module")
def lib():
    from streaming_sparse_b200 import build
    build.build()
    from streaming_sparse_b200._lib import lib as load
    return load()


def test_host_argument_errors(lib):
    fake = ctypes.c_void_p(0x100000)  # never dereferenced: every call fails its host checks, or has no rows
    odd = ctypes.c_void_p(0x100002)
    q = lib.ss_quant_rows
    assert q(fake, 64, 0, 0, 64, fake, 64, fake, None) == 0
    assert q(fake, 63, 0, 4, 64, fake, 64, fake, None) == 1001      # rows overlap
    assert q(fake, 64, 3, 4, 64, fake, 64, fake, None) == 1001      # no such type
    assert q(fake, 64, 0, 4, 0, fake, 64, fake, None) == 1001
    assert q(None, 64, 0, 4, 64, fake, 64, fake, None) == 1002
    assert q(odd, 64, 1, 4, 64, fake, 64, fake, None) == 1002       # fp32 off 4 bytes
    r = lib.ss_rms_norm_i8
    assert r(fake, 64, None, 0, 0, 0, 64, fake, 1e-6, None, 0, fake, 64, fake, None) == 0
    assert r(fake, 64, None, 0, 0, 4, 64, None, 1e-6, None, 0, fake, 64, fake, None) == 1002
    assert r(fake, 64, fake, 32, 0, 4, 64, fake, 1e-6, None, 0, fake, 64, fake, None) == 1001
    a = lib.ss_adaln_i8
    tail = (1e-6, None, 0, fake, 64, fake, None)
    assert a(fake, 64, None, 0, None, 0, 0, 0, 64, 4, fake, fake, 64, None, None, *tail) == 0
    assert a(fake, 64, None, 0, None, 0, 0, 4, 64, 4, None, None, 0, None, None, *tail) == 1001   # neither form
    assert a(fake, 64, None, 0, None, 0, 0, 4, 64, 4, fake, fake, 64, fake, fake, *tail) == 1001  # both
    assert a(fake, 64, None, 0, None, 0, 0, 4, 64, 0, fake, fake, 64, None, None, *tail) == 1001  # no frame size
    assert a(fake, 64, None, 0, fake, 64, 0, 4, 64, 4, fake, fake, 64, None, None, *tail) == 1002  # a gate without y
    assert a(fake, 64, None, 0, None, 0, 0, 4, 64, 4, fake, None, 64, None, None, *tail) == 1002
    g = lib.ss_linear_i8
    assert g(fake, 64, fake, fake, 64, fake, None, 0, 0, 0, 8, 64, fake, 8, 0, None, None) == 0
    assert g(fake, 64, fake, fake, 64, fake, None, 0, 0, 4, 0, 64, fake, 8, 0, None, None) == 1001
    assert g(fake, 72, fake, fake, 64, fake, None, 0, 0, 4, 8, 64, fake, 8, 0, None, None) == 1001   # stride off 16
    assert g(fake, 131072, fake, fake, 131072, fake, None, 0, 0, 4, 8, 131072, fake, 8, 0, None, None) == 1001
    assert g(fake, 64, fake, fake, 64, fake, fake, 3, 0, 4, 8, 64, fake, 8, 0, None, None) == 1001
    assert g(odd, 64, fake, fake, 64, fake, None, 0, 0, 4, 8, 64, fake, 8, 0, None, None) == 1002
    assert g(fake, 64, fake, fake, 64, None, None, 0, 0, 4, 8, 64, fake, 8, 0, None, None) == 1002
    assert g(fake, 64, fake, fake, 64, fake, None, 0, 0, 4, 8, 64, odd, 8, 1, None, None) == 1002


def test_host_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q, s = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: ops.quant_rows(x), lambda: ops.rms_norm_i8(x, x[0], 1e-6),
                 lambda: ops.adaln_i8(x, eps=1e-6, weight=x[0], bias=x[0]), lambda: ops.linear_i8(q, s, q, s)):
        with pytest.raises(ValueError):
            call()


def test_rows_i8_start_at_multiples_of_16_bytes():
    for d in (1, 15, 16, 17, 1536, 1549):
        t = ops.rows_i8(3, d, "cpu")
        assert t.shape == (3, d) and t.stride(1) == 1 and t.stride(0) % 16 == 0 and t.stride(0) >= d


class NoLibrary:
    """Stands in for the library: a call that should have been refused before it fails the test."""

    def __getattr__(self, name):
        def called(*args):
            pytest.fail(f"{name} was called")
        return called


@pytest.fixture()
def cuda_tensors(monkeypatch):
    """CUDA tensors without memory or a GPU, device 0 current, and no library."""
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0)
    monkeypatch.setattr(ops, "lib", lambda: NoLibrary())
    with FakeTensorMode():
        yield


def test_tensors_of_another_device_than_the_current_are_refused(cuda_tensors):
    dev = torch.device("cuda:1")
    x, w = torch.empty(4, 64, dtype=torch.bfloat16, device=dev), torch.empty(64, dtype=torch.bfloat16, device=dev)
    q, s = torch.empty(4, 64, dtype=torch.int8, device=dev), torch.empty(4, device=dev)
    for call in (lambda: ops.quant_rows(x), lambda: ops.rms_norm_i8(x, w, 1e-6),
                 lambda: ops.adaln_i8(x, eps=1e-6, weight=w, bias=w), lambda: ops.linear_i8(q, s, q, s)):
        with pytest.raises(ValueError, match="current device"):
            call()


def test_sizes_past_32_bits_are_refused(cuda_tensors):
    """The library's sizes are 32-bit integers: larger ones would reach it as their low bits."""
    dev, big = torch.device("cuda:0"), 2 ** 32 + 64
    for shape in ((1, big), (big, 1)):
        x, w = torch.empty(shape, dtype=torch.bfloat16, device=dev), torch.empty(shape[1], dtype=torch.bfloat16, device=dev)
        for call in (lambda: ops.quant_rows(x), lambda: ops.rms_norm_i8(x, w, 1e-6),
                     lambda: ops.adaln_i8(x, eps=1e-6, weight=w, bias=w)):
            with pytest.raises(ValueError, match="at most"):
                call()
    q, s = torch.empty(big, 16, dtype=torch.int8, device=dev), torch.empty(big, device=dev)
    with pytest.raises(ValueError, match="at most"):
        ops.linear_i8(q, s, q[:8], s[:8])
    with pytest.raises(ValueError, match="at most"):
        ops.linear_i8(q[:8], s[:8], q, s)


def test_tensors_with_a_tangent_are_refused():
    """Forward-mode derivatives would be lost without a word: under no_grad() too, which does not stop them."""
    x = torch.randn(4, 8)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                with pytest.raises(ValueError, match="forward-mode"):
                    ops._no_grad(None, x, dual)
                ops._no_grad(x, None, torch.autograd.forward_ad.unpack_dual(dual).primal)
    ops._no_grad(x, None)
    with pytest.raises(ValueError, match="forward-mode"):
        torch.func.jvp(lambda v: ops._no_grad(v) or v, (x,), (torch.ones_like(x),))


@pytest.mark.gpu
def test_calls_inside_a_dual_level():
    dev = torch.device("cuda:0")
    x, w = torch.randn(4, 64, device=dev), torch.ones(64, device=dev)
    em = torch.randn(1, 2, 64, device=dev)
    q, s = ops.quant_rows(x)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.quant_rows(dual(x)), lambda: ops.rms_norm_i8(dual(x), w, 1e-6),
                     lambda: ops.rms_norm_i8(x, dual(w), 1e-6), lambda: ops.rms_norm_i8(x, w, 1e-6, residual=dual(x)),
                     lambda: ops.adaln_i8(x, eps=1e-6, weight=w, bias=dual(w)),
                     lambda: ops.adaln_i8(x, eps=1e-6, shift=dual(em[:, 0]), scale=em[:, 1], frame_tokens=4),
                     lambda: ops.linear_i8(q, dual(s), q, s), lambda: ops.linear_i8(q, s, q, s, bias=dual(s))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        assert torch.equal(ops.quant_rows(x)[0], q)


def test_a_timeout_says_whose_it_is():
    for name, text in (("timeout", "attention"), ("linear_timeout", "8-bit linear")):
        word = ops.DeviceStatus.word("cpu")
        word.fill_(ops.DEV_BITS[name])
        with pytest.raises(RuntimeError, match=text) as e:
            ops.DeviceStatus.check("cpu")
        assert len([t for t in ("attention", "8-bit linear") if t in str(e.value)]) == 1 and not word.any()
    assert len(set(ops.DEV_BITS.values())) == len(ops.DEV_BITS)
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "ssparse.h")) as f:
        header = {n: int(v, 16) for n, v in re.findall(r"#define SS_DEV_(\w+) (0x\w+)", f.read())}
    assert header == {n.upper(): v for n, v in ops.DEV_BITS.items()}
