"""Argument checks of the 8-bit layer's C entry points and host operators (no GPU: nothing is launched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from triattention_amd.kernels import linear as Q
from triattention_amd.kernels.extension import Module, load_library

FAKE = ctypes.c_void_p(4096)  # aligned, never dereferenced: validation fails before any launch
ODD = ctypes.c_void_p(4104)


def refused(call, text):
    lib = load_library()
    assert call(lib) != 0
    assert text in lib.tri_last_error(), lib.tri_last_error()


def test_row_quantizers_check_their_arguments():
    rows = lambda **c: lambda lib: lib.tri_quantize_rows(*(dict(  # noqa: E731
        x=FAKE, ldx=64, dtype=1, m=4, k=64, codes=FAKE, ldc=64, scales=FAKE, stream=None) | c).values())
    refused(rows(x=None), b"null buffer")
    refused(rows(codes=None), b"null buffer")
    refused(rows(scales=None), b"null buffer")
    refused(rows(dtype=3), b"dtype")
    refused(rows(k=0), b"1 to 2^31")
    refused(rows(m=-1), b"1 to 2^31")
    refused(rows(ldc=63), b"may not overlap")
    refused(rows(ldx=-64), b"row strides")
    norm = lambda **c: lambda lib: lib.tri_rms_norm_quant(*(dict(  # noqa: E731
        x=FAKE, ldx=64, residual=FAKE, ldr=64, weight=FAKE, dtype=1, m=4, k=64, eps=1e-6, codes=FAKE, ldc=64,
        scales=FAKE, hidden=FAKE, ldh=64, stream=None) | c).values())
    refused(norm(weight=None), b"null buffer")
    refused(norm(hidden=None), b"both or neither")
    refused(norm(residual=None), b"both or neither")
    refused(norm(ldh=10), b"may not overlap")
    for eps in (0.0, -1e-6, float("nan"), float("inf"), 1e-60):
        refused(norm(eps=eps), b"eps must be positive")
    refused(lambda lib: lib.tri_silu_mul_quant(FAKE, 64, None, 64, 1, 4, 64, FAKE, 64, FAKE, None), b"null buffer")


def test_products_check_their_arguments():
    call = lambda **c: lambda lib: lib.tri_int8_linear(*(dict(  # noqa: E731
        x=FAKE, ldx=64, xs=FAKE, w=FAKE, ldw=64, ws=FAKE, bias=None, residual=None, ldr=0, out=FAKE, ldo=32, dtype=1,
        m=4, n=32, k=64, workspace=None, bytes=0, stream=None) | c).values())
    for name in ("x", "xs", "w", "ws", "out"):
        refused(call(**{name: None}), b"null buffer")
    refused(call(x=ODD), b"16-byte aligned")
    refused(call(w=ODD), b"16-byte aligned")
    refused(call(ldx=68), b"16-byte aligned")
    refused(call(ldw=8), b"16-byte aligned")
    refused(call(ldx=(1 << 22) + 16), b"at most 4 MiB")
    refused(call(ldx=-64), b"at most 4 MiB")
    refused(call(k=131072), b"at most 131071")
    refused(call(k=0), b"empty shape")
    refused(call(n=0), b"empty shape")
    refused(call(m=(1 << 30) + 1), b"2^30")
    refused(call(ldo=31), b"may not overlap")
    refused(call(dtype=-1), b"dtype")
    refused(lambda lib: lib.tri_int8_linear_workspace(1, 1, 1, None), b"null output")


def test_no_rows_need_no_buffers():
    lib = load_library()
    assert lib.tri_quantize_rows(None, 64, 1, 0, 64, None, 64, None, None) == 0
    assert lib.tri_rms_norm_quant(None, 64, None, 0, None, 1, 0, 64, 1e-6, None, 64, None, None, 0, None) == 0
    assert lib.tri_silu_mul_quant(None, 64, None, 64, 1, 0, 64, None, 64, None, None) == 0
    assert lib.tri_int8_linear(None, 64, None, None, 64, None, None, None, 0, None, 32, 1, 0, 32, 64, None, 0, None) == 0


class _NoLaunch(Module):
    """The binding with its launches recorded instead of made."""

    def __init__(self):
        super().__init__(load_library())
        self.calls = []

    def _launch_for(self, x, fn, *args):
        self.calls.append((fn.__name__, args))

    def int8_linear_workspace(self, m, n, k, device):
        return 0


@pytest.fixture
def module(monkeypatch):
    found = _NoLaunch()
    monkeypatch.setattr(Q, "load_extension", lambda: found)
    return found


def test_codes_rows_start_at_multiples_of_16_bytes(module):
    for k in (1, 15, 16, 17, 100, 128):
        codes, scales = Q.quantize_rows(torch.ones(3, k))
        assert codes.shape == (3, k) and codes.stride(0) % 16 == 0 and codes.stride(0) - k < 16
        assert scales.shape == (3,)
    codes, scales, h = Q.rms_norm_quant(torch.ones(2, 3, 20), torch.ones(20), 1e-5, residual=torch.ones(2, 3, 20))
    assert codes.shape == h.shape == (2, 3, 20) and scales.shape == (2, 3)
    out = Q.int8_linear(codes, scales, *Q.quantize_rows(torch.ones(7, 20)))
    assert out.shape == (2, 3, 7) and out.dtype == torch.bfloat16


def test_host_operators_refuse(module):
    x = torch.ones(2, 3, 20)
    codes, scales = Q.quantize_rows(x)
    w, ws = Q.quantize_rows(torch.ones(7, 20))
    seen = len(module.calls)
    bad = [lambda: Q.quantize_rows(x.transpose(0, 1)), lambda: Q.quantize_rows(x.double()),
           lambda: Q.quantize_rows(torch.ones(())), lambda: Q.quantize_rows(x.clone().requires_grad_()),
           lambda: Q.rms_norm_quant(x, torch.ones(19), 1e-6), lambda: Q.rms_norm_quant(x, torch.ones(20).half(), 1e-6),
           lambda: Q.rms_norm_quant(x, torch.ones(20), 1e-6, residual=torch.ones(6, 20)),
           lambda: Q.silu_mul_quant(x, x[:1]), lambda: Q.silu_mul_quant(x, x.half()),
           lambda: Q.int8_linear(codes, scales[0], w, ws), lambda: Q.int8_linear(codes, scales, w[:, :19], ws),
           lambda: Q.int8_linear(codes, scales, w, ws[:6]), lambda: Q.int8_linear(codes, scales, w.float(), ws),
           lambda: Q.int8_linear(codes, scales, w, ws, bias=torch.ones(7)),
           lambda: Q.int8_linear(codes, scales, w, ws, residual=torch.ones(2, 3, 7)),
           lambda: Q.int8_linear(codes, scales, w, ws, residual=torch.ones(6, 7).bfloat16()),
           lambda: Q.int8_linear(codes, scales, w, ws, out_dtype=torch.float64),
           lambda: Q.int8_linear(codes, scales.requires_grad_(), w, ws)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    assert len(module.calls) == seen
    with torch.no_grad():
        Q.quantize_rows(x.clone().requires_grad_())  # (nothing asks for the gradient here)
