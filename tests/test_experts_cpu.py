"""What the experts' computation refuses, through the C ABI and through the package: contracts are checked before anything touches a GPU."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, FP8, I32, F32 = 1, 2, 4, 6


class Tensor(ctypes.Structure):
    _fields_ = [('data', ctypes.c_void_p), ('dtype', ctypes.c_int32), ('ndim', ctypes.c_int32), ('size', ctypes.c_int64 * 2),
                ('stride', ctypes.c_int64 * 2)]


def matrix(rows, cols, dtype=BF16, ld=None, col=1, at=4096):
    return Tensor(at, dtype, 2, (ctypes.c_int64 * 2)(rows, cols), (ctypes.c_int64 * 2)(cols if ld is None else ld, col))


def vector(n, dtype, at=4096, stride=1):
    return Tensor(at, dtype, 1, (ctypes.c_int64 * 2)(n, 0), (ctypes.c_int64 * 2)(stride, 0))


class Linear(ctypes.Structure):
    _fields_ = [(n, Tensor) for n in ('x', 'x_sf', 'weight', 'weight_sf', 'psum', 'out')] + [
        ('weight_expert_stride', ctypes.c_int64), ('weight_sf_expert_stride', ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ('num_experts', 'expert_alignment', 'zero_rows', 'transpose_weight')] + [('stream', ctypes.c_void_p)]


class WeightGrad(ctypes.Structure):
    _fields_ = [(n, Tensor) for n in ('grad', 'x', 'psum', 'out')] + [('out_expert_stride', ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ('num_experts', 'expert_alignment', 'accumulate')] + [('stream', ctypes.c_void_p)]


class Swiglu(ctypes.Structure):
    _fields_ = [(n, Tensor) for n in ('h', 'weights', 'psum', 'out', 'out_sf')] + [
        (n, ctypes.c_int32) for n in ('num_experts', 'expert_alignment', 'zero_rows')] + [('stream', ctypes.c_void_p)]


class SwigluGrad(ctypes.Structure):
    _fields_ = [(n, Tensor) for n in ('grad', 'h', 'weights', 'psum', 'grad_h', 'grad_weights')] + [
        (n, ctypes.c_int32) for n in ('num_experts', 'expert_alignment', 'zero_rows')] + [('stream', ctypes.c_void_p)]


@pytest.fixture(scope='module')
def lib():
    import deep_ep
    lib = deep_ep._C._lib
    for name in ('ep_grouped_linear', 'ep_grouped_weight_grad', 'ep_swiglu', 'ep_swiglu_grad'):
        getattr(lib, name).restype = ctypes.c_int
        getattr(lib, name).argtypes = [ctypes.c_void_p]
    lib.ep_last_error.restype = ctypes.c_char_p
    return lib


def refused(lib, name, args):
    assert getattr(lib, name)(ctypes.addressof(args)) != 0
    message = lib.ep_last_error().decode()
    assert message.startswith('Assertion exception (ep_experts.cpp:'), message
    return message


def linear(fp8=False, **changes):
    t = FP8 if fp8 else BF16
    values = dict(x=matrix(64, 256, t), weight=matrix(128, 256, t), psum=vector(4, I32), out=matrix(64, 128), weight_expert_stride=128 * 256,
                  num_experts=4, expert_alignment=16)
    if fp8:
        values.update(x_sf=matrix(64, 2, F32), weight_sf=matrix(1, 2, F32), weight_sf_expert_stride=2)
    values.update(changes)
    a = Linear()
    for k, v in values.items():
        setattr(a, k, v)
    return a


LINEAR = {
    'rows that are not contiguous': dict(x=matrix(64, 256, col=2, ld=512)),
    'rows off 16 bytes': dict(x=matrix(64, 256, ld=257)),
    'a pointer off 16 bytes': dict(x=matrix(64, 256, at=4098)),
    'overlapping rows': dict(x=matrix(64, 256, ld=128)),
    'float32 rows': dict(x=matrix(64, 256, F32)),
    'mixed types': dict(weight=matrix(128, 256, FP8)),
    'another depth': dict(weight=matrix(128, 264)),
    'odd depth': dict(x=matrix(64, 252, ld=256), weight=matrix(128, 252, ld=256)),
    'odd columns': dict(weight=matrix(124, 256), out=matrix(64, 124, ld=128)),
    'a psum of another length': dict(psum=vector(5, I32)),
    'a psum of 64 bits': dict(psum=vector(4, 5)),
    'a strided psum': dict(psum=vector(4, I32, stride=2)),
    'no psum for several experts': dict(psum=Tensor()),
    'no experts': dict(num_experts=0),
    'no alignment': dict(expert_alignment=0),
    'unknown zero_rows': dict(zero_rows=3),
    'a result of other rows': dict(out=matrix(63, 128)),
    'a float32 result': dict(out=matrix(64, 128, F32)),
    'experts off 16 bytes': dict(weight_expert_stride=128 * 256 + 4),
    'scales of bfloat16 rows': dict(x_sf=matrix(64, 2, F32)),
    'too many rows': dict(x=matrix(2 ** 31, 256), out=matrix(2 ** 31, 128)),
    'rows of many megabytes': dict(x=matrix(64, 256, ld=2 ** 22)),
    'no rows tensor': dict(x=Tensor()),
}
LINEAR_FP8 = {
    'no scales': dict(x_sf=Tensor()),
    'no weight scales': dict(weight_sf=Tensor()),
    'scales of too few groups': dict(x_sf=matrix(64, 1, F32)),
    'weight scales of too few blocks': dict(weight_sf=matrix(1, 1, F32)),
    'scales in bfloat16': dict(x_sf=matrix(64, 2, BF16)),
    'transposed weights': dict(transpose_weight=1, x=matrix(64, 128, FP8), x_sf=matrix(64, 1, F32), out=matrix(64, 256)),
    'depth off 16 channels': dict(x=matrix(64, 248, FP8, ld=256), weight=matrix(128, 248, FP8, ld=256)),
    'depth beyond the table of scales': dict(x=matrix(64, 32896, FP8), weight=matrix(128, 32896, FP8), x_sf=matrix(64, 257, F32),
                                             weight_sf=matrix(1, 257, F32)),
}


@pytest.mark.parametrize('case', LINEAR)
def test_grouped_linear_refuses(lib, case):
    refused(lib, 'ep_grouped_linear', linear(**LINEAR[case]))


@pytest.mark.parametrize('case', LINEAR_FP8)
def test_grouped_linear_of_fp8_refuses(lib, case):
    refused(lib, 'ep_grouped_linear', linear(fp8=True, **LINEAR_FP8[case]))


@pytest.mark.parametrize('change', [
    dict(x=matrix(63, 256)), dict(grad=matrix(64, 128, FP8)), dict(grad=matrix(64, 124, ld=128)), dict(out=matrix(128, 248, ld=256)),
    dict(out=matrix(128, 256, 5)), dict(accumulate=1), dict(out_expert_stride=128 * 256 - 8), dict(num_experts=3), dict(psum=Tensor())])
def test_grouped_weight_grad_refuses(lib, change):
    a = WeightGrad()
    values = dict(grad=matrix(64, 128), x=matrix(64, 256), psum=vector(4, I32), out=matrix(128, 256), out_expert_stride=128 * 256,
                  num_experts=4, expert_alignment=16)
    for k, v in {**values, **change}.items():
        setattr(a, k, v)
    refused(lib, 'ep_grouped_weight_grad', a)


@pytest.mark.parametrize('change', [
    dict(h=matrix(64, 504)), dict(h=matrix(64, 512, F32)), dict(out=matrix(64, 248)), dict(out=matrix(64, 256, FP8)),
    dict(out_sf=matrix(64, 2, F32)), dict(out=matrix(64, 256, FP8), out_sf=matrix(64, 3, F32)), dict(weights=vector(63, F32)),
    dict(weights=vector(64, F32, stride=2)), dict(weights=vector(64, BF16)), dict(expert_alignment=-1), dict(zero_rows=-1)])
def test_swiglu_refuses(lib, change):
    a = Swiglu()
    values = dict(h=matrix(64, 512), psum=vector(4, I32), out=matrix(64, 256), num_experts=4, expert_alignment=16)
    for k, v in {**values, **change}.items():
        setattr(a, k, v)
    refused(lib, 'ep_swiglu', a)


@pytest.mark.parametrize('change', [
    dict(grad=matrix(64, 248)), dict(grad=matrix(63, 256)), dict(grad_h=matrix(64, 256)), dict(grad_h=matrix(64, 512, F32)),
    dict(grad_weights=vector(64, BF16)), dict(grad_weights=vector(65, F32)), dict(num_experts=2)])
def test_swiglu_grad_refuses(lib, change):
    a = SwigluGrad()
    values = dict(grad=matrix(64, 256), h=matrix(64, 512), psum=vector(4, I32), grad_h=matrix(64, 512), num_experts=4, expert_alignment=16)
    for k, v in {**values, **change}.items():
        setattr(a, k, v)
    refused(lib, 'ep_swiglu_grad', a)


def test_missing_arguments_are_refused(lib):
    for name in ('ep_grouped_linear', 'ep_grouped_weight_grad', 'ep_swiglu', 'ep_swiglu_grad'):
        assert getattr(lib, name)(None) != 0


def test_tensors_of_the_host_are_refused():
    import deep_ep
    x, w, psum = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(1, 8, 16, dtype=torch.bfloat16), torch.tensor([4], dtype=torch.int32)
    with pytest.raises(deep_ep._C.EPException, match='must live on the GPU'):
        deep_ep.grouped_linear(x, w, (psum, 1))
    with pytest.raises(deep_ep._C.EPException, match='must live on the GPU'):
        deep_ep.swiglu(x, (psum, 1))
    with pytest.raises(deep_ep._C.EPException, match='must live on the GPU'):
        deep_ep.grouped_linear_grad(torch.zeros(4, 8, dtype=torch.bfloat16), x, w, (psum, 1))


def test_what_has_no_gradient_is_refused():
    import deep_ep
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16, requires_grad=True), torch.zeros(8, 16, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match='gradients'):
        deep_ep.grouped_linear(x, w, out=torch.zeros(4, 8, dtype=torch.bfloat16))
    with pytest.raises(AssertionError, match='gradients'):
        deep_ep.grouped_linear((torch.zeros(4, 16).to(torch.float8_e4m3fn), torch.ones(4, 1, requires_grad=True)), w)
    with pytest.raises(AssertionError, match='gradients'):
        deep_ep.swiglu(x, fused_fp8_quant=True)
    with pytest.raises(AssertionError, match='pair'):
        deep_ep.swiglu(x.detach(), out=torch.zeros(4, 8, dtype=torch.bfloat16), fused_fp8_quant=True)
