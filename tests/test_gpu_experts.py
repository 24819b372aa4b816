"""The experts' computation on the GPU against plain sums in 64 bits."""
import pytest
import torch

import deep_ep
import experts_util as U

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'

# counts of the experts, alignment, rows behind the last expert's
LAYOUTS = {
    'one_row': ([1], 1, 0),
    'empty_first_and_last': ([0, 5, 0, 0, 17, 1, 0], 16, 3),
    'ragged': ([129, 1, 0, 64, 255, 3], 128, 0),
    'unaligned': ([33, 7, 0, 130, 2], 1, 5),
    'odd_alignment': ([33, 7, 0, 130, 2], 24, 0),
    'none': ([0, 0, 0], 8, 4),
    'long': ([300, 513, 0, 40], 64, 100),
    'many_experts': ([(i * 7) % 5 for i in range(161)], 4, 0),
}
# depth, columns: below, at and above the steps of 64 and 128 channels and tiles of 128 and 256, odd multiples of eight
SIZES = [(8, 8), (64, 128), (72, 136), (256, 512), (264, 72), (1000, 264)]


def _dev(t):
    return tuple(x.to(DEV) for x in t) if isinstance(t, tuple) else t.to(DEV)


def _sentinel(*shape, dtype=torch.bfloat16):
    return torch.full(shape, 77.0, dtype=dtype, device=DEV)


def _check_rows(got, layout, zeroed, sentinel=None):
    got = got.cpu()
    if zeroed:
        assert (got[layout.padding] == 0).all()
    rest = ~layout.valid & ~layout.padding if zeroed else ~layout.valid
    if sentinel is not None:
        assert (got[rest] == sentinel).all(), 'rows of no expert were written'


@pytest.mark.parametrize('name', LAYOUTS)
@pytest.mark.parametrize('depth,columns', SIZES)
@pytest.mark.parametrize('fp8', [False, True])
def test_grouped_linear(name, depth, columns, fp8):
    if fp8:
        depth = -(-depth // 16) * 16
    layout = U.Layout(*LAYOUTS[name])
    x = U.normal(1, layout.rows, depth)
    w = U.normal(2, len(layout.counts), columns, depth, scale=depth ** -0.5)
    more = torch.zeros((layout.rows, 1))
    if fp8:
        x, w = U.quantise_rows(x), U.quantise_weights(w)
        want, size = U.linear(x, w, layout)
        more = U.fp8_error(x, w, layout)
        x[0].view(torch.uint8)[~layout.valid] = 0x7f
        U.spoil(x[1], layout)
    else:
        want, size = U.linear(x, w, layout)
        U.spoil(x, layout)
    for zeroed in (False, True):
        out = _sentinel(layout.rows, columns)
        y = deep_ep.grouped_linear(_dev(x), _dev(w), layout.on(DEV), out=out, do_zero_padding=zeroed)
        assert y.data_ptr() == out.data_ptr()
        U.assert_sum(y[layout.valid.to(DEV)], want[layout.valid], size[layout.valid], depth, what=name, more=more[layout.valid])
        _check_rows(y, layout, zeroed, 77.0)
    y = deep_ep.grouped_linear(_dev(x), _dev(w), layout.on(DEV), do_zero_padding=True)
    assert torch.equal(y[layout.valid.to(DEV)], out[layout.valid.to(DEV)])
    _check_rows(y, layout, True)


@pytest.mark.parametrize('name', LAYOUTS)
@pytest.mark.parametrize('depth,columns', SIZES)
def test_grouped_linear_gradients(name, depth, columns):
    layout = U.Layout(*LAYOUTS[name])
    x = U.spoil(U.normal(1, layout.rows, depth), layout)
    w = U.normal(2, len(layout.counts), columns, depth, scale=depth ** -0.5)
    grad = U.spoil(U.normal(3, layout.rows, columns), layout)
    want_x, size_x = U.linear(torch.nan_to_num(grad), w.transpose(1, 2), layout)
    want_w, size_w = U.weight_grad(torch.nan_to_num(grad), torch.nan_to_num(x), layout)
    dx, dw, dg = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), grad.to(DEV)
    y = deep_ep.grouped_linear(dx, dw, layout.on(DEV), do_zero_padding=True)
    y.backward(dg)
    U.assert_sum(dx.grad, want_x, size_x, columns, what='rows')      # (all of them: rows of no expert have a gradient of zero)
    most = max(layout.counts)
    U.assert_sum(dw.grad, want_w, size_w, most, what='weights')
    gx, none = deep_ep.grouped_linear_grad(dg, dx.detach(), dw.detach(), layout.on(DEV), need_weight=False)
    assert none is None and torch.equal(gx[layout.valid.to(DEV)], dx.grad[layout.valid.to(DEV)])
    # into the caller's float32 gradients, which hold something
    held = U.normal(4, *w.shape).float()
    total = held.to(DEV)
    none, gw = deep_ep.grouped_linear_grad(dg, dx.detach(), dw.detach(), layout.on(DEV), need_x=False, grad_weight=total, accumulate=True)
    assert none is None and gw.data_ptr() == total.data_ptr()
    U.assert_sum(total, want_w + held.double(), size_w + held.double().abs(), most, half=2.0 ** -24, what='accumulated')
    deep_ep.grouped_linear_grad(dg, dx.detach(), dw.detach(), layout.on(DEV), need_x=False, grad_weight=total)
    U.assert_sum(total, want_w, size_w, most, half=2.0 ** -24, what='float32')


def test_gradients_agree_with_differences():
    """Along a direction, in 64 bits on the CPU: what the formulas of the gradients are held to is the derivative of the forward formula."""
    layout = U.Layout([3, 0, 6], 4)
    x, w = U.normal(1, layout.rows, 16).double(), U.normal(2, 3, 8, 16).double()
    grad, tx, tw = U.normal(3, layout.rows, 8).double(), U.normal(4, layout.rows, 16).double(), U.normal(5, 3, 8, 16).double()
    f = lambda t: (U.linear(x + t * tx, w + t * tw, layout)[0] * grad)[layout.valid].sum()  # noqa: E731
    gx, gw = U.linear(grad, w.transpose(1, 2), layout)[0], U.weight_grad(grad, x, layout)[0]
    h = 1e-4
    assert abs((f(h) - f(-h)) / (2 * h) - ((gx * tx)[layout.valid].sum() + (gw * tw).sum())) < 1e-6


def _swiglu(h, w):
    gate, up = h.double().chunk(2, dim=1)
    return gate * torch.sigmoid(gate) * up * (1.0 if w is None else w.double()[:, None])


# exponential, reciprocal and six products and sums in 32 bits, each a unit in the last place off at most; the exponential's argument too,
# which a gate up to 2^7 turns into 2^7 times its relative error
SWIGLU_ERROR = (8 + 2 ** 7) * 2.0 ** -23


@pytest.mark.parametrize('name', LAYOUTS)
@pytest.mark.parametrize('channels', [8, 72, 128, 520, 2048])
@pytest.mark.parametrize('weighted', [False, True])
def test_swiglu(name, channels, weighted):
    layout = U.Layout(*LAYOUTS[name])
    h = U.normal(1, layout.rows, 2 * channels, scale=3.0)
    w = torch.rand(layout.rows, generator=torch.Generator().manual_seed(2)) if weighted else None
    want = _swiglu(h, w)[layout.valid]
    h = U.spoil(h, layout).to(DEV)
    if weighted:
        w = U.spoil(w, layout).to(DEV)
    valid = layout.valid.to(DEV)
    for zeroed in (False, True):
        out = _sentinel(layout.rows, channels)
        deep_ep.swiglu(h, layout.on(DEV), w, out=out, do_zero_padding=zeroed)
        error = (out[valid].cpu().double() - want).abs() - want.abs() * (U.HALF_BF16 + 2 * SWIGLU_ERROR) - 1e-38
        assert error.numel() == 0 or error.max() <= 0
        _check_rows(out, layout, zeroed, 77.0)
        q, sf = _sentinel(layout.rows, channels).to(torch.float8_e4m3fn), _sentinel(layout.rows, -(-channels // 128), dtype=torch.float32)
        held = q[:1, :1].float().cpu().item() if layout.rows else 0.0
        deep_ep.swiglu(h, layout.on(DEV), w, fused_fp8_quant=True, out=(q, sf), do_zero_padding=zeroed)
        amax = torch.nn.functional.pad(want.abs(), (0, -channels % 128)).unflatten(1, (-(-channels // 128), 128)).amax(dim=2).clamp(1e-4)
        got_sf = sf[valid].cpu().double()
        assert ((got_sf - amax / 448).abs() <= amax / 448 * (SWIGLU_ERROR + 2.0 ** -23)).all()
        value = U.widen_rows((q[valid].cpu(), sf[valid].cpu()))
        # half a step of e4m3 (2^-4 of the value; 2^-10 of a scale below the normal range), behind the value's own error
        error = (value - want).abs() - (want.abs() * (2.0 ** -4 + 2 * SWIGLU_ERROR)
                                        + got_sf.repeat_interleave(128, 1)[:, :channels] * 2.0 ** -10 * 1.001)
        assert error.numel() == 0 or error.max() <= 0
        _check_rows(q.float(), layout, zeroed, held)
        _check_rows(sf, layout, zeroed, 77.0)


@pytest.mark.parametrize('name', LAYOUTS)
@pytest.mark.parametrize('channels', [8, 136, 520, 2048])
@pytest.mark.parametrize('weighted', [False, True])
def test_swiglu_gradients(name, channels, weighted):
    layout = U.Layout(*LAYOUTS[name])
    h = U.normal(1, layout.rows, 2 * channels, scale=3.0)
    w = torch.rand(layout.rows, generator=torch.Generator().manual_seed(2)) if weighted else None
    grad = U.normal(3, layout.rows, channels)
    ref_h = h.double()[layout.valid].requires_grad_()
    ref_w = w.double()[layout.valid].requires_grad_() if weighted else None
    _swiglu(ref_h, ref_w).backward(grad.double()[layout.valid])
    dh = U.spoil(h.clone(), layout).to(DEV).requires_grad_()
    dw = U.spoil(w.clone(), layout).to(DEV).requires_grad_() if weighted else None
    y = deep_ep.swiglu(dh, layout.on(DEV), dw, do_zero_padding=True)
    y.backward(U.spoil(grad.clone(), layout).to(DEV))
    assert (dh.grad.cpu()[~layout.valid] == 0).all()
    gate, up = h.double()[layout.valid].chunk(2, dim=1)
    g = grad.double()[layout.valid].abs() * (1.0 if w is None else w.double()[layout.valid][:, None])
    # (1 + gate (1 - sigmoid)) may cancel: its error is that of its terms
    size = torch.cat([g * up.abs() * torch.sigmoid(gate) * (1 + gate.abs()), g * (gate * torch.sigmoid(gate)).abs()], dim=1)
    got = dh.grad.cpu().double()[layout.valid]
    error = (got - ref_h.grad).abs() - (ref_h.grad.abs() * U.HALF_BF16 + size * 2 * SWIGLU_ERROR + 1e-38)
    assert error.numel() == 0 or error.max() <= 0
    if weighted:
        assert dw.grad.dtype == torch.float32 and (dw.grad.cpu()[~layout.valid] == 0).all()
        terms = (grad.double()[layout.valid] * _swiglu(h[layout.valid], None)).abs().sum(dim=1)
        assert ((dw.grad.cpu().double()[layout.valid] - ref_w.grad).abs() <= terms * (2 * SWIGLU_ERROR + channels * 2.0 ** -23)).all()


def test_swiglu_at_the_ends_of_the_range():
    """Large gates either way, infinities and NaN: a row keeps its own to itself."""
    h = torch.zeros((4, 16), dtype=torch.bfloat16)
    h[0, :8] = torch.tensor([-3e38, -200.0, -90.0, -1.0, 0.0, 1.0, 90.0, 3e4])
    h[0, 8:] = 2.0
    h[1], h[2, :8], h[2, 8:], h[3, 3] = float('nan'), float('inf'), 1.0, float('-inf')
    want = _swiglu(h, None)
    got = deep_ep.swiglu(h.to(DEV)).cpu().double()
    assert torch.equal(torch.isnan(got[1]), torch.isnan(want[1])) and torch.isinf(got[2]).all()
    # the exponential of gates beyond -88 has no float32: the value, below 1e-36, comes out as zero
    assert ((got[0] - want[0]).abs() <= want[0].abs() * 2.0 ** -7 + 1e-35).all()
    q, sf = deep_ep.swiglu(h.to(DEV), fused_fp8_quant=True)
    assert torch.isnan(q[1].float()).all() and torch.isfinite(q[0].float()).all() and torch.isfinite(sf[0]).all()
