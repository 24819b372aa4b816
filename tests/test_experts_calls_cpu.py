"""Calls of the experts' computation that the package refuses before anything touches a GPU."""
import pytest
import torch

import deep_ep

REFUSED = 'a result must not lie on an operand'
ELSEWHERE = 'must live on the GPU'      # what a call of host tensors that nothing else is wrong with ends with


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _ends_with(message, call, *args, **kwargs):
    with pytest.raises(deep_ep._C.EPException, match=message):
        call(*args, **kwargs)


# columns of x and of the result in one buffer of 8 x 256
@pytest.mark.parametrize('x,out,message', [
    ((0, 64), (0, 64), REFUSED), ((0, 64), (32, 96), REFUSED), ((32, 96), (0, 64), REFUSED), ((64, 128), (120, 184), REFUSED),
    ((0, 64), (64, 128), ELSEWHERE), ((192, 256), (0, 64), ELSEWHERE), ((0, 64), (192, 256), ELSEWHERE)])
def test_columns_of_one_matrix(x, out, message):
    wide = _bf16(8, 256)
    x, out = wide[:, slice(*x)], wide[:, slice(*out)]
    _ends_with(message, deep_ep.grouped_linear, x, _bf16(64, 64), out=out)
    _ends_with(message, deep_ep.grouped_linear, x[3:], _bf16(64, 64), out=out[:5])
    idx = torch.zeros(8, dtype=torch.int32)
    _ends_with(message, deep_ep.grouped_lora_linear, x, _bf16(64, 64), _bf16(1, 8, 64), _bf16(1, 64, 8), idx, out=out)
    _ends_with(message, deep_ep.swiglu, x, out=out)      # (of other columns too: shapes are looked at behind this)


def test_rows_of_one_matrix():
    wide = _bf16(16, 64)
    w = _bf16(64, 64)
    _ends_with(REFUSED, deep_ep.grouped_linear, wide[:8], w, out=wide[7:15])
    _ends_with(REFUSED, deep_ep.grouped_linear, wide[0::2], w, out=wide[0:8])
    _ends_with(ELSEWHERE, deep_ep.grouped_linear, wide[:8], w, out=wide[8:])
    _ends_with(ELSEWHERE, deep_ep.grouped_linear, wide[0::2], w, out=wide[1::2])
    _ends_with(ELSEWHERE, deep_ep.grouped_linear, wide[:0], w, out=wide[:0])


def test_every_operand_is_looked_at():
    layout, idx = (torch.tensor([8, 16], dtype=torch.int32), 8), torch.zeros(16, dtype=torch.int32)
    wide = _bf16(2, 16, 96)
    x, out = _bf16(16, 64), wide[0, :, :16]
    _ends_with(REFUSED, deep_ep.grouped_linear, x, wide[:, :, 8:72], layout, out=out)
    _ends_with(ELSEWHERE, deep_ep.grouped_linear, x, wide[:, :, 16:80], layout, out=out)
    _ends_with(REFUSED, deep_ep.grouped_linear, x, _bf16(2, 16, 64), (out.view(torch.int32)[:1].reshape(-1)[:2], 8), out=out)
    a, b = _bf16(3, 2, 8, 96), _bf16(3, 2, 16, 24)
    _ends_with(REFUSED, deep_ep.grouped_lora_linear, x, _bf16(2, 16, 64), a[..., :64], b[..., :8], idx, layout, out=a[0].view(16, 96)[:, 48:64])
    _ends_with(REFUSED, deep_ep.grouped_lora_linear, x, _bf16(2, 16, 64), a[..., :64], b[..., :8], idx, layout, out=b[1, 1, :, :16])
    _ends_with(ELSEWHERE, deep_ep.grouped_lora_linear, x, _bf16(2, 16, 64), a[..., :64], b[..., :8], idx, layout, out=b[1, 1, :, 8:])
    # fp8 rows with their scales behind them, the results of swiglu side by side
    packed = torch.zeros(16, 64 + 16, dtype=torch.uint8)
    q, sf = packed[:, :64].view(torch.float8_e4m3fn), packed[:, 64:68].view(torch.float32)
    w = (_bf16(16, 64).to(torch.float8_e4m3fn), torch.zeros(1, 1))
    bytes_ = packed.view(torch.bfloat16)
    _ends_with(REFUSED, deep_ep.grouped_linear, (q, sf), w, out=torch.as_strided(bytes_, (16, 16), (40, 1), 24))
    _ends_with(ELSEWHERE, deep_ep.swiglu, _bf16(16, 128), fused_fp8_quant=True, out=(q, sf))
    _ends_with(REFUSED, deep_ep.swiglu, _bf16(16, 128), fused_fp8_quant=True, out=(q, packed[:, 60:64].view(torch.float32)))
    h = _bf16(16, 192)
    weights = h.view(torch.float32)[:, 64:65].reshape(-1)
    _ends_with(REFUSED, deep_ep.swiglu, h[:, :128], None, weights, out=h[:, 128:])      # (the weights are its first two columns)
    _ends_with(ELSEWHERE, deep_ep.swiglu, h[:, :64], None, weights, out=h[:, 136:168])
    shared = torch.zeros(64)
    _ends_with(REFUSED, deep_ep.swiglu, _bf16(16, 16), None, shared[:16], out=shared.view(torch.bfloat16).view(16, 8))


def test_gradients_of_weights_and_their_operands():
    wide = _bf16(64, 256)
    grad, x = wide[:, :64], wide[:, 64:128]
    for at, message in ((0, REFUSED), (32, REFUSED), (120, REFUSED), (128, ELSEWHERE), (192, ELSEWHERE)):
        _ends_with(message, deep_ep.grouped_linear_grad, grad, x, _bf16(64, 64), need_x=False, grad_weight=wide[:, at:at + 64])


def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad
    layout, idx = (torch.tensor([4], dtype=torch.int32), 1), torch.zeros(4, dtype=torch.int32)
    x, w, a, b, scales = _bf16(4, 64), _bf16(1, 64, 64), _bf16(1, 1, 8, 64), _bf16(1, 1, 64, 8), torch.ones(1)
    grad, q, qw = _bf16(4, 64), (_bf16(4, 64).to(torch.float8_e4m3fn), torch.ones(4, 1)), (_bf16(1, 64, 64).to(torch.float8_e4m3fn), torch.ones(1, 1, 1))
    message = 'forward-mode gradients are not implemented'
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        _ends_with(message, deep_ep.grouped_linear, dual(x), w, layout)
        _ends_with(message, deep_ep.grouped_linear, x, dual(w), layout)
        _ends_with(message, deep_ep.grouped_linear, dual(x.detach().requires_grad_()), w, layout)
        _ends_with(message, deep_ep.grouped_linear, (q[0], dual(q[1])), qw, layout)
        _ends_with(message, deep_ep.grouped_linear, q, (qw[0], dual(qw[1])), layout)
        _ends_with(message, deep_ep.grouped_linear_grad, dual(grad), x, w, layout)
        _ends_with(message, deep_ep.grouped_linear_grad, grad, x, dual(w), layout, need_weight=False)
        _ends_with(message, deep_ep.grouped_linear_grad, grad, dual(x), w, layout, need_x=False)
        _ends_with(message, deep_ep.swiglu, dual(x), layout)
        _ends_with(message, deep_ep.swiglu, x, layout, dual(torch.ones(4)))
        _ends_with(message, deep_ep.swiglu_grad, grad[:, :32], dual(x), layout)
        _ends_with(message, deep_ep.swiglu_grad, grad[:, :32], x, layout, dual(torch.ones(4)))
        _ends_with(message, deep_ep.grouped_lora_linear, dual(x), w, a, b, idx, layout)
        _ends_with(ELSEWHERE, deep_ep.grouped_linear, x, w, layout)
    with torch.no_grad(), forward_ad.dual_level():
        _ends_with(message, deep_ep.grouped_linear, forward_ad.make_dual(x, x), w, layout)


def test_results_with_a_gradient_of_their_own_are_refused():
    """Such a tensor's graph would not know of the value that is stored into it."""
    x, w, h = _bf16(4, 64), _bf16(64, 64), _bf16(4, 128)
    a, b, idx = _bf16(1, 8, 64), _bf16(1, 64, 8), torch.zeros(4, dtype=torch.int32)
    leaf = _bf16(4, 64).requires_grad_()
    for out in (leaf, leaf * 2):
        for call, *args in ((deep_ep.grouped_linear, x, w), (deep_ep.swiglu, h), (deep_ep.grouped_lora_linear, x, w, a, b, idx)):
            with pytest.raises(AssertionError, match='gradients'):
                call(*args, out=out)
            with torch.no_grad():
                _ends_with(ELSEWHERE, call, *args, out=out)
        with pytest.raises(AssertionError, match='gradients'):
            deep_ep.grouped_linear_grad(x, x, _bf16(4, 64), need_x=False, grad_weight=out)
    with pytest.raises(AssertionError, match='gradients'):
        deep_ep.swiglu(h, fused_fp8_quant=True, out=(_bf16(4, 64).to(torch.float8_e4m3fn), torch.zeros(4, 1, requires_grad=True)))


@pytest.mark.parametrize('stride,ok', [((0, 1), False), ((0, 0), False), ((1, 0), False), ((1, 63), False), ((1, 1), False), ((-2, 1), False),
                                       ((2, 1), True), ((1, 64), True), ((1, 80), True), ((5, 2), True)])
def test_scales_that_lie_on_each_other_are_refused(stride, ok):
    """Scales that swiglu stores, [64, 2]: every one has a place of its own."""
    import ctypes
    import test_experts_cpu as C
    lib = deep_ep._C._lib
    a = C.Swiglu()
    sf = C.matrix(64, 2, C.F32)
    sf.stride[0], sf.stride[1] = stride
    for k, v in dict(h=C.matrix(64, 512), psum=C.vector(4, C.I32), out=C.matrix(64, 256, C.FP8), out_sf=sf, num_experts=4, expert_alignment=16).items():
        setattr(a, k, v)
    lib.ep_swiglu.argtypes = [ctypes.c_void_p]
    if torch.cuda.is_available() and ok:
        pytest.skip('the addresses are not memory')
    assert lib.ep_swiglu(ctypes.addressof(a)) != 0
    lib.ep_last_error.restype = ctypes.c_char_p
    message = lib.ep_last_error().decode()
    # (what is right comes as far as the missing GPU)
    assert message.startswith('Assertion exception (ep_experts.cpp:') != ok, message
