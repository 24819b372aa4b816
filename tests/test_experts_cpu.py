"""What the experts' computation refuses, through the C ABI and through the package: contracts are checked before anything touches a GPU."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, FP8, I32, F32 = 1, 2, 4, 6
ENTRIES = ('ep_grouped_linear', 'ep_grouped_lora_linear', 'ep_grouped_weight_grad', 'ep_swiglu', 'ep_swiglu_grad')


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
        (n, ctypes.c_int32) for n in ('num_experts', 'expert_alignment', 'zero_rows', 'transpose_weight')] + [
        ('workspace', ctypes.c_void_p), ('workspace_bytes', ctypes.c_int64), ('stream', ctypes.c_void_p)]


class WeightGrad(ctypes.Structure):
    _fields_ = [(n, Tensor) for n in ('grad', 'x', 'psum', 'out')] + [('out_expert_stride', ctypes.c_int64)] + [
        (n, ctypes.c_int32) for n in ('num_experts', 'expert_alignment', 'accumulate')] + [
        ('workspace', ctypes.c_void_p), ('workspace_bytes', ctypes.c_int64), ('stream', ctypes.c_void_p)]


class Swiglu(ctypes.Structure):
    _fields_ = [(n, Tensor) for n in ('h', 'weights', 'psum', 'out', 'out_sf')] + [
        (n, ctypes.c_int32) for n in ('num_experts', 'expert_alignment', 'zero_rows')] + [('stream', ctypes.c_void_p)]


class SwigluGrad(ctypes.Structure):
    _fields_ = [(n, Tensor) for n in ('grad', 'h', 'weights', 'psum', 'grad_h', 'grad_weights')] + [
        (n, ctypes.c_int32) for n in ('num_experts', 'expert_alignment', 'zero_rows')] + [('stream', ctypes.c_void_p)]


class Lora(ctypes.Structure):
    _fields_ = [('linear', Linear)] + [(n, Tensor) for n in ('lora_a', 'lora_b', 'adapter_idx', 'scales')] + [
        (n, ctypes.c_int64) for n in ('a_adapter', 'a_expert', 'b_adapter', 'b_expert')] + [
        ('num_adapters', ctypes.c_int32), ('reserved', ctypes.c_int32), ('workspace', ctypes.c_void_p), ('workspace_bytes', ctypes.c_int64)]


@pytest.fixture(scope='module')
def lib():
    import deep_ep
    lib = deep_ep._C._lib
    for name in ENTRIES:
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
    'a workspace of no address': dict(workspace_bytes=16),
    'a workspace off 16 bytes': dict(workspace=4104, workspace_bytes=16),
    'a workspace of less than nothing': dict(workspace=4096, workspace_bytes=-1),
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
    dict(out=matrix(128, 256, 5)), dict(accumulate=1), dict(out_expert_stride=128 * 256 - 8), dict(num_experts=3), dict(psum=Tensor()),
    dict(workspace_bytes=64), dict(workspace=4100, workspace_bytes=64), dict(workspace=4096, workspace_bytes=-4)])
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
    for name in ENTRIES:
        assert getattr(lib, name)(None) != 0
    assert lib.ep_expand_token_index(None, None, None, None, None) != 0


def lora(**changes):
    values = dict(linear=linear(), lora_a=matrix(16, 256), lora_b=matrix(128, 16), adapter_idx=vector(64, I32), a_adapter=4 * 16 * 256,
                  a_expert=16 * 256, b_adapter=4 * 128 * 16, b_expert=128 * 16, num_adapters=3, workspace=4096, workspace_bytes=1 << 30)
    values.update(changes)
    a = Lora()
    for k, v in values.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize('change', [
    dict(linear=linear(fp8=True)), dict(linear=linear(x=matrix(64, 128), out=matrix(64, 256), transpose_weight=1)),
    dict(lora_a=matrix(16, 248, ld=256)), dict(lora_a=matrix(12, 256), lora_b=matrix(128, 12, ld=16)),
    dict(lora_a=matrix(72, 256), lora_b=matrix(128, 72)), dict(lora_b=matrix(120, 16)), dict(lora_b=matrix(128, 8)),
    dict(lora_a=matrix(16, 256, F32)), dict(num_adapters=0), dict(a_adapter=4), dict(b_expert=-8), dict(adapter_idx=vector(63, I32)),
    dict(adapter_idx=vector(64, 5)), dict(adapter_idx=Tensor()), dict(scales=vector(2, F32)), dict(scales=vector(3, BF16)),
    dict(workspace=None), dict(workspace=4100), dict(workspace_bytes=64 * 16 * 4 - 1)])
def test_grouped_lora_refuses(lib, change):
    refused(lib, 'ep_grouped_lora_linear', lora(**change))


def test_lora_workspace(lib):
    f = lib.ep_grouped_lora_workspace_bytes
    f.restype, f.argtypes = ctypes.c_int64, [ctypes.c_int64, ctypes.c_int, ctypes.c_int64, ctypes.c_int]
    for bad in ((-1, 1, 64, 8), (4, 0, 64, 8), (4, 1, 0, 8), (4, 1, 64, 0), (4, 1, 64, 72)):
        assert f(*bad) == -1
    assert f(0, 1, 64, 8) == 0
    for rows in (1, 7, 61, 500, 3000, 100000):
        for experts in (1, 8, 160):
            for depth in (8, 512, 520, 7168):
                chunks, rest = divmod(f(rows, experts, depth, 16), rows * 16 * 4)
                assert rest == 0 and 1 <= chunks <= 16 and chunks <= -(-depth // 512)


@pytest.mark.parametrize('change', [dict(values=vector(8, 5)), dict(metadata=matrix(8, 2, I32)), dict(metadata=vector(8, I32)), dict(psum=vector(0, I32)),
                                    dict(psum=Tensor()), dict(out=vector(16, F32)), dict(out=vector(16, I32, stride=2))])
def test_expand_token_index_refuses(lib, change):
    a = {**dict(values=vector(8, I32), metadata=matrix(8, 4, I32), psum=vector(1, I32), out=vector(16, I32)), **change}
    f = lib.ep_expand_token_index
    f.argtypes = [ctypes.c_void_p] * 5
    assert f(*(ctypes.addressof(a[k]) for k in ('values', 'metadata', 'psum', 'out')), None) != 0
    assert lib.ep_last_error().decode().startswith('Assertion exception (ep_experts.cpp:')


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
    with pytest.raises(AssertionError, match='gradients'):
        deep_ep.grouped_lora_linear(x, w, w[None], w[None], torch.zeros(4, dtype=torch.int32))
    with pytest.raises(AssertionError, match='pair'):
        deep_ep.swiglu(x.detach(), out=torch.zeros(4, 8, dtype=torch.bfloat16), fused_fp8_quant=True)


def test_code_object_is_built_with_its_kernels():
    import deep_ep
    path = os.path.join(os.path.dirname(deep_ep.__file__), 'lib', 'ep_experts.hsaco')
    with open(path, 'rb') as f:
        data = f.read()
    assert b'gfx950' in data
    for name in ('ep_grouped_bf16_256x256', 'ep_grouped_fp8_64x256', 'ep_grouped_transposed_128x256', 'ep_grouped_lora_32x64', 'ep_grouped_split_lora_64',
                 'ep_grouped_weights_f32_256x256', 'ep_lora_down_rows', 'ep_sum_splits', 'ep_swiglu_fp8', 'ep_swiglu_gradients', 'ep_expand_token_index_rows'):
        assert name.encode() in data, name
