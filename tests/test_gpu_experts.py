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


# mean rows of an expert on both sides of the lines between tiles, tails of every size in them
@pytest.mark.parametrize('counts', [[700, 0, 190, 513], [257, 383, 128, 64, 1], [160, 161, 90], [40, 47, 48, 49, 16], [5000], [9000, 9100, 7],
                                    [97] * 40, [3, 80, 1, 0] * 40])
@pytest.mark.parametrize('depth,columns', [(16, 520), (1008, 776), (2048, 256)])
@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'lora', 'gradients'])
def test_every_tile(counts, depth, columns, kind):
    layout = U.Layout(counts, 16)
    experts = len(counts)
    x, w = U.normal(1, layout.rows, depth), U.normal(2, experts, columns, depth, scale=depth ** -0.5)
    v = layout.valid
    if kind == 'gradients':
        grad = U.normal(3, layout.rows, columns)
        gx, gw = deep_ep.grouped_linear_grad(_dev(grad), _dev(x), _dev(w), layout.on(DEV))
        want, size = U.linear(grad, w.transpose(1, 2), layout)
        U.assert_sum(gx[v.to(DEV)], want[v], size[v], columns, what='rows')
        U.assert_sum(gw, *U.weight_grad(grad, x, layout), max(counts), what='weights')
        return
    if kind == 'lora':
        a, b = U.normal(4, 5, experts, 24, depth, scale=depth ** -0.5), U.normal(5, 5, experts, columns, 24)
        idx = (torch.arange(layout.rows) // 37 % 7 - 1).to(torch.int32)
        want, size, low = _lora(x, w, a, b, None, idx, layout)
        y = deep_ep.grouped_lora_linear(_dev(x), _dev(w), _dev(a), _dev(b), _dev(idx), layout.on(DEV))
        U.assert_sum(y[v.to(DEV)], want[v], size[v], depth, more=(low * (2.0 ** -17 + (depth + 40) * U.STEP_F32))[v])
        return
    more = torch.zeros((layout.rows, 1))
    if kind == 'fp8':
        x, w = U.quantise_rows(x), U.quantise_weights(w)
        more = U.fp8_error(x, w, layout)
    want, size = U.linear(x, w, layout)
    y = deep_ep.grouped_linear(_dev(x), _dev(w), layout.on(DEV))
    U.assert_sum(y[v.to(DEV)], want[v], size[v], depth, more=more[v])


@pytest.mark.parametrize('counts,alignment', [([1], 1), ([61], 1), ([0, 130, 3], 16), ([9, 0, 0, 2, 30, 1, 1, 5], 8)])
@pytest.mark.parametrize('depth,columns', [(1536, 136), (7168, 512), (7120, 264)])
@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'lora'])
def test_depth_in_parts(counts, alignment, depth, columns, kind):
    """Few tiles: the depth is split, the parts are added in a launch of their own."""
    layout = U.Layout(counts, alignment, tail=3)
    experts = len(counts)
    lib, c64 = deep_ep._C._lib, deep_ep._C.ctypes.c_int64
    in_parts = lib.ep_grouped_linear_workspace_bytes(c64(layout.rows), experts, alignment, c64(depth), c64(columns), int(kind == 'lora')) > 0
    assert in_parts == (kind == 'lora' or depth > 7000)
    x, w = U.normal(1, layout.rows, depth), U.normal(2, experts, columns, depth, scale=depth ** -0.5)
    a, b = U.normal(4, 3, experts, 8, depth, scale=depth ** -0.5), U.normal(5, 3, experts, columns, 8)
    idx = (torch.arange(layout.rows) % 4 - 1).to(torch.int32)
    v = layout.valid
    more = torch.zeros((layout.rows, 1))
    if kind == 'fp8':
        x, w = U.quantise_rows(x), U.quantise_weights(w)
        more = U.fp8_error(x, w, layout)
    if kind == 'lora':
        want, size, low = _lora(x, w, a, b, None, idx, layout)
        more = low * (2.0 ** -17 + (depth + 40) * U.STEP_F32)
    else:
        want, size = U.linear(x, w, layout)
    U.spoil(x[1] if kind == 'fp8' else x, layout)
    for zeroed in (False, True):
        out = _sentinel(layout.rows, columns)
        if kind == 'lora':
            deep_ep.grouped_lora_linear(_dev(x), _dev(w), _dev(a), _dev(b), _dev(idx), layout.on(DEV), out=out, do_zero_padding=zeroed)
        else:
            deep_ep.grouped_linear(_dev(x), _dev(w), layout.on(DEV), out=out, do_zero_padding=zeroed)
        U.assert_sum(out[v.to(DEV)], want[v], size[v], depth, more=more[v])
        _check_rows(out, layout, zeroed, 77.0)


@pytest.mark.parametrize('counts', [[5000], [2100, 0, 1700]])
@pytest.mark.parametrize('rows,columns', [(72, 136), (256, 512)])
def test_weight_gradients_of_rows_in_parts(counts, rows, columns):
    layout = U.Layout(counts, 16)
    experts = len(counts)
    lib, c64 = deep_ep._C._lib, deep_ep._C.ctypes.c_int64
    assert lib.ep_grouped_weight_grad_workspace_bytes(c64(layout.rows), experts, 16, c64(rows), c64(columns)) > 0
    grad, x = U.spoil(U.normal(1, layout.rows, rows), layout), U.spoil(U.normal(2, layout.rows, columns), layout)
    w = torch.zeros(experts, rows, columns, dtype=torch.bfloat16, device=DEV)
    want, size = U.weight_grad(torch.nan_to_num(grad), torch.nan_to_num(x), layout)
    _, gw = deep_ep.grouped_linear_grad(_dev(grad), _dev(x), w, layout.on(DEV), need_x=False)
    U.assert_sum(gw, want, size, max(counts))
    held = U.normal(4, experts, rows, columns).float()
    wide = torch.zeros(experts, rows + 8, columns + 8, device=DEV)
    total = wide[:, 8:, 8:]
    total.copy_(held)
    deep_ep.grouped_linear_grad(_dev(grad), _dev(x), w, layout.on(DEV), need_x=False, grad_weight=total, accumulate=True)
    U.assert_sum(total, want + held.double(), size + held.double().abs(), max(counts), half=2.0 ** -24)
    assert (wide[:, :8] == 0).all() and (wide[:, :, :8] == 0).all()


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


def _lora_inputs(layout, adapters, rank, depth, columns, shared, seed=5):
    experts = len(layout.counts)
    x, w = U.normal(seed, layout.rows, depth), U.normal(seed + 1, experts, columns, depth, scale=depth ** -0.5)
    a = U.normal(seed + 2, adapters, experts, rank, depth, scale=depth ** -0.5)
    b = U.normal(seed + 3, adapters, experts, columns, rank)
    scales = torch.rand(adapters, generator=torch.Generator().manual_seed(seed + 4)) + 0.5
    return x, w, a, b, scales


def _lora(x, w, a, b, scales, idx, layout):
    """Values, and what the tolerance counts: the product's magnitudes, and the adapters' part's with both of its sums."""
    y, size = U.linear(x, w, layout)
    low_size = torch.zeros_like(y)
    for e, mine in enumerate(layout.slices()):
        for n in range(a.size(0)):
            rows = torch.arange(layout.rows)[mine][idx[mine] == n]
            s = 1.0 if scales is None else scales[n].double()
            y[rows] += s * (x[rows].double() @ a[n, e].double().t()) @ b[n, e].double().t()
            low_size[rows] += s * (x[rows].double().abs() @ a[n, e].double().abs().t()) @ b[n, e].double().abs().t()
    return y, size, low_size


@pytest.mark.parametrize('name', LAYOUTS)
@pytest.mark.parametrize('adapters,rank,depth,columns', [(1, 8, 8, 8), (3, 16, 264, 136), (40, 40, 1032, 72), (7, 64, 520, 264)])
@pytest.mark.parametrize('mixed', [False, True])
def test_grouped_lora(name, adapters, rank, depth, columns, mixed):
    layout = U.Layout(*LAYOUTS[name])
    x, w, a, b, scales = _lora_inputs(layout, adapters, rank, depth, columns, False)
    gen = torch.Generator().manual_seed(9)
    # any order, or in runs as requests have it; numbers of no adapter on either side
    idx = torch.randint(-1, adapters + 1, (layout.rows,), generator=gen) if mixed else \
        torch.arange(layout.rows) * (adapters + 2) // max(1, layout.rows) - 1
    idx = idx.to(torch.int32)
    scales = scales if mixed else None
    want, size, low = _lora(x, w, a, b, scales, idx, layout)
    idx[~layout.valid] = 0
    U.spoil(x, layout)
    out = _sentinel(layout.rows, columns)
    deep_ep.grouped_lora_linear(_dev(x), _dev(w), _dev(a), _dev(b), _dev(idx), layout.on(DEV), scales=None if scales is None else _dev(scales), out=out)
    # the low-rank rows are sums in 32 bits too, handed on as two BF16 that keep 2^-17 of them
    more = low * (2.0 ** -17 + (depth + rank + 16) * U.STEP_F32)
    v = layout.valid
    U.assert_sum(out[v.to(DEV)], want[v], size[v], depth, what=name, more=more[v])
    _check_rows(out, layout, False, 77.0)


@pytest.mark.parametrize('rows', [0, 1, 17, 61, 300, 2300])
def test_lora_beside_a_shared_projection(rows):
    layout = U.Layout([rows], 1)
    x, w, a, b, scales = _lora_inputs(layout, 5, 16, 1024, 256, True)
    idx = torch.randint(0, 5, (rows,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    want, size, low = _lora(x, w, a, b, scales, idx, layout)
    y = deep_ep.grouped_lora_linear(_dev(x), _dev(w[0]), _dev(a[:, 0]), _dev(b[:, 0]), _dev(idx), scales=_dev(scales))
    U.assert_sum(y, want, size, 1024, more=low * (2.0 ** -17 + 2048 * U.STEP_F32))
    # without adapters it is the product alone
    none = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    y = deep_ep.grouped_lora_linear(_dev(x), _dev(w[0]), _dev(a[:, 0]), _dev(b[:, 0]), none)
    U.assert_sum(y, *U.linear(x, w[:1], U.Layout([rows], 1)), 1024)


@pytest.mark.parametrize('rows,columns', [(40, 256), (700, 1024), (5000, 256), (5000, 2048)])
@pytest.mark.parametrize('value', [float('inf'), float('nan')])
def test_an_adapter_that_is_not_finite_stays_with_its_rows(rows, columns, value):
    layout = U.Layout([rows], 1)
    x, w, a, b, _ = _lora_inputs(layout, 3, 16, 512, columns, True)
    idx = (torch.arange(rows) % 4 - 1).to(torch.int32)
    want, size, low = _lora(x, w, a, b, None, idx, layout)
    b[1, 0, 77, 3] = value
    y = deep_ep.grouped_lora_linear(_dev(x), _dev(w[0]), _dev(a[:, 0]), _dev(b[:, 0]), _dev(idx))
    more = (low * (2.0 ** -17 + 1024 * U.STEP_F32)).expand(size.shape)
    hers = torch.zeros(size.shape, dtype=torch.bool)
    hers[idx == 1, 77] = True
    assert not torch.isfinite(y.cpu()[hers]).any()
    U.assert_sum(y.cpu()[~hers], want[~hers], size[~hers], 512, more=more[~hers])
    # the first matrix: a row's low-rank row is infinite or NaN, and all of its result
    a[2, 0, 5, 100] = value
    y = deep_ep.grouped_lora_linear(_dev(x), _dev(w[0]), _dev(a[:, 0]), _dev(b[:, 0]), _dev(idx)).cpu()
    hers[idx == 2] = True
    assert not torch.isfinite(y[hers]).any()
    U.assert_sum(y[~hers], want[~hers], size[~hers], 512, more=more[~hers])


def test_two_calls_at_once():
    """On two streams, each with its workspaces."""
    x, w = _dev(U.normal(1, 64, 7168)), [_dev(U.normal(2 + i, 512, 7168)) for i in range(2)]
    a, b, idx = _dev(U.normal(4, 2, 16, 7168)), _dev(U.normal(5, 2, 512, 16)), (torch.arange(64, dtype=torch.int32) % 2).to(DEV)
    want = [deep_ep.grouped_lora_linear(x, m, a, b, idx) for m in w]
    grads = [deep_ep.grouped_linear_grad(want[0], x, m)[0] for m in w]
    streams, got = [torch.cuda.Stream() for _ in w], [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, m, g in zip(streams, w, got):
            with torch.cuda.stream(s):
                g.append((deep_ep.grouped_lora_linear(x, m, a, b, idx), deep_ep.grouped_linear_grad(want[0], x, m)[0]))
    torch.cuda.synchronize()
    for i in range(2):
        for y, g in got[i]:
            assert torch.equal(y, want[i]) and torch.equal(g, grads[i])


def test_adapters_as_views():
    """Matrices of adapters and experts inside larger tensors, and one that all adapters share."""
    layout = U.Layout([20, 3, 40], 8)
    x, w, a, b, scales = _lora_inputs(layout, 4, 16, 128, 64, False)
    idx = torch.randint(-1, 4, (layout.rows,), generator=torch.Generator().manual_seed(2)).to(torch.int32)
    want = deep_ep.grouped_lora_linear(_dev(x), _dev(w), _dev(a), _dev(b), _dev(idx), layout.on(DEV), do_zero_padding=True)
    wide_a, wide_b = torch.zeros(3, 4, 24, 136, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 3, 64, 40, dtype=torch.bfloat16, device=DEV)
    va, vb = wide_a.transpose(0, 1)[:, :, 8:, :128], wide_b[..., 8:24]
    va.copy_(a), vb.copy_(b)
    wide_x = torch.zeros(layout.rows, 256, dtype=torch.bfloat16, device=DEV)
    vx = wide_x[:, 64:192]
    vx.copy_(x)
    wide_w = torch.zeros(64, 3, 128, dtype=torch.bfloat16, device=DEV)
    vw = wide_w.transpose(0, 1)
    vw.copy_(w)
    got = deep_ep.grouped_lora_linear(vx, vw, va, vb, _dev(idx), layout.on(DEV), do_zero_padding=True)
    assert torch.equal(got, want)
    one = deep_ep.grouped_lora_linear(_dev(x), _dev(w), _dev(a[1:2].expand(4, -1, -1, -1).contiguous()), _dev(b), _dev(idx), layout.on(DEV), do_zero_padding=True)
    same = deep_ep.grouped_lora_linear(_dev(x), _dev(w), _dev(a)[1:2].expand(4, -1, -1, -1), _dev(b), _dev(idx), layout.on(DEV), do_zero_padding=True)
    assert torch.equal(one, same)


def test_views_of_rows_scales_and_results():
    layout = U.Layout([70, 0, 9], 16, 5)
    x, w = U.quantise_rows(U.normal(1, layout.rows, 320)), U.quantise_weights(U.normal(2, 3, 136, 320))
    want = deep_ep.grouped_linear(_dev(x), _dev(w), layout.on(DEV), do_zero_padding=True)
    # scales by columns, as a dispatch with use_tma_aligned_col_major_sf returns them; weights' scales transposed; a slice of a wider result
    columns = _dev(x[1]).t().contiguous().t()
    scales = _dev(w[1]).transpose(1, 2).contiguous().transpose(1, 2)
    wide = _sentinel(layout.rows, 200)
    deep_ep.grouped_linear((_dev(x[0]), columns), (_dev(w[0]), scales), layout.on(DEV), out=wide[:, 32:168], do_zero_padding=True)
    covered = (layout.valid | layout.padding).to(DEV)
    assert torch.equal(wide[covered, 32:168], want[covered])
    assert (wide[:, :32] == 77).all() and (wide[:, 168:] == 77).all() and (wide[~covered] == 77).all()
    h = _dev(U.normal(3, layout.rows, 512))
    a, (q, sf) = deep_ep.swiglu(h, layout.on(DEV), do_zero_padding=True), deep_ep.swiglu(h, layout.on(DEV), fused_fp8_quant=True, do_zero_padding=True)
    wide_h = torch.zeros(layout.rows, 1024, dtype=torch.bfloat16, device=DEV)
    wide_h[:, 256:768] = h
    by_columns = torch.zeros(2, layout.rows, device=DEV).t()
    wide_q = torch.zeros(layout.rows, 264, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    deep_ep.swiglu(wide_h[:, 256:768], layout.on(DEV), fused_fp8_quant=True, out=(wide_q[:, 8:], by_columns), do_zero_padding=True)
    assert torch.equal(wide_q[:, 8:].float()[covered], q.float()[covered]) and torch.equal(by_columns[covered], sf[covered])
    assert torch.equal(deep_ep.swiglu(wide_h[:, 256:768], layout.on(DEV), do_zero_padding=True)[covered], a[covered])


def test_offsets_past_32_bits():
    """Rows 4 MiB apart, experts 4 GiB apart: what contiguous tensors give, to the last bit."""
    layout = U.Layout([700, 0, 400], 1)
    rows, experts, ld, far = layout.rows, 3, 2 << 20, (2 << 30) + 64
    big = [torch.empty(rows * ld, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    wide = torch.empty(experts * far, dtype=torch.bfloat16, device=DEV)

    def put(buffer, t):
        return buffer.as_strided(t.shape, (ld, 1)).copy_(t)
    x, w, h = _dev(U.normal(1, rows, 256)), _dev(U.normal(2, experts, 128, 256)), _dev(U.normal(3, rows, 512))
    vw = wide.as_strided(w.shape, (far, 256, 1)).copy_(w)
    vx, out = put(big[0], x), big[1].as_strided((rows, 128), (ld, 1))
    psum = layout.on(DEV)
    want = deep_ep.grouped_linear(x, w, psum)
    assert torch.equal(deep_ep.grouped_linear(vx, vw, psum, out=out), want)
    gx, gw = deep_ep.grouped_linear_grad(want, x, w, psum)
    a, b = _dev(U.normal(4, 2, experts, 16, 256)), _dev(U.normal(5, 2, experts, 128, 16))
    idx = (torch.arange(rows, dtype=torch.int32) % 3 - 1).to(DEV)
    lora = deep_ep.grouped_lora_linear(x, w, a, b, idx, psum)
    assert torch.equal(deep_ep.grouped_lora_linear(vx, vw, a, b, idx, psum, out=out), lora)
    out.copy_(want)
    vgx, vgw = deep_ep.grouped_linear_grad(out, vx, vw, psum, grad_weight=vw)
    assert torch.equal(vgx, gx) and torch.equal(vgw, gw)
    one = deep_ep.grouped_linear(x[:40], w[0])
    assert torch.equal(deep_ep.grouped_linear(vx[-40:].copy_(x[:40]), vw[2].copy_(w[0]), out=out[-40:]), one)
    vh, out = put(big[0], h), big[1].as_strided((rows, 256), (ld, 1))
    assert torch.equal(deep_ep.swiglu(vh, psum, out=out), deep_ep.swiglu(h, psum))
    assert torch.equal(deep_ep.swiglu_grad(out, vh, psum)[0], deep_ep.swiglu_grad(deep_ep.swiglu(h, psum), h, psum)[0])


def test_counts_beyond_the_tensors_stay_inside():
    """Whatever the counts say, no row outside the tensors is touched (an expert that ends behind the last row ends with it)."""
    x, w = _dev(U.normal(1, 40, 64)), _dev(U.normal(2, 3, 32, 64))
    wide = _sentinel(104, 32)
    psum = torch.tensor([30, 200, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    deep_ep.grouped_linear(x, w, (psum, 16), out=wide[32:72], do_zero_padding=True)
    assert (wide[:32] == 77).all() and (wide[72:] == 77).all()
    want = deep_ep.grouped_linear(x, w, (torch.tensor([30, 40, 40], dtype=torch.int32, device=DEV), 16), do_zero_padding=True)
    assert torch.equal(wide[32:72], want)
    deep_ep.swiglu(x, (psum, 16), out=wide[32:72])
    assert (wide[:32] == 77).all() and (wide[72:] == 77).all()
    negative = torch.tensor([-5, -(2 ** 31), 7], dtype=torch.int32, device=DEV)
    deep_ep.grouped_linear(x, w, (negative, 16), out=wide[32:72])
    deep_ep.swiglu(x, (negative, 16), out=wide[32:72])
    deep_ep.grouped_linear_grad(_dev(U.normal(3, 40, 32)), x, w, (psum, 16))
    assert (wide[:32] == 77).all() and (wide[72:] == 77).all()


def test_broadcast_gradients():
    layout = U.Layout([5, 20], 8)
    x, w = _dev(U.normal(1, layout.rows, 64)).requires_grad_(), _dev(U.normal(2, 2, 32, 64)).requires_grad_()
    y = deep_ep.grouped_linear(x, w, layout.on(DEV), do_zero_padding=True)
    y.sum().backward()                                   # a gradient of one value, broadcast
    gx, gw = deep_ep.grouped_linear_grad(torch.ones_like(y), x.detach(), w.detach(), layout.on(DEV), do_zero_padding=True)
    assert torch.equal(x.grad, gx) and torch.equal(w.grad, gw)
    h = _dev(U.normal(3, layout.rows, 64)).requires_grad_()
    a = deep_ep.swiglu(h, layout.on(DEV), do_zero_padding=True)
    a.t().contiguous().t().sum(dim=0).sum().backward()
    assert torch.equal(h.grad, deep_ep.swiglu_grad(torch.ones_like(a), h.detach(), layout.on(DEV), do_zero_padding=True)[0])


def test_gradients_of_some_arguments_only():
    layout = U.Layout([5, 20], 8)
    x, w, h, g = _dev(U.normal(1, layout.rows, 64)), _dev(U.normal(2, 2, 32, 64)), _dev(U.normal(3, layout.rows, 64)), torch.rand(layout.rows, device=DEV)
    grad = _dev(U.normal(4, layout.rows, 32))
    gx, gw = deep_ep.grouped_linear_grad(grad, x, w, layout.on(DEV), do_zero_padding=True)
    for with_x in (True, False):
        lx, lw = x.detach().requires_grad_(with_x), w.detach().requires_grad_(not with_x)
        deep_ep.grouped_linear(lx, lw, layout.on(DEV)).backward(grad)
        assert torch.equal(lx.grad, gx) and lw.grad is None if with_x else torch.equal(lw.grad, gw) and lx.grad is None
    gh, gg = deep_ep.swiglu_grad(grad, h, layout.on(DEV), g, do_zero_padding=True)
    for with_h in (True, False):
        lh, lg = h.detach().requires_grad_(with_h), g.detach().requires_grad_(not with_h)
        deep_ep.swiglu(lh, layout.on(DEV), lg).backward(grad)
        assert torch.equal(lh.grad, gh) and lg.grad is None if with_h else torch.equal(lg.grad, gg) and lh.grad is None


def test_gradients_are_not_differentiated():
    x, w = _dev(U.normal(1, 8, 64)).requires_grad_(), _dev(U.normal(2, 32, 64)).requires_grad_()
    y = deep_ep.grouped_linear(x, w)
    gx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='cannot be differentiated'):
        gx.float().pow(2).sum().backward()
    h = _dev(U.normal(3, 8, 64)).requires_grad_()
    gh, = torch.autograd.grad(deep_ep.swiglu(h).sum(), h, create_graph=True)
    with pytest.raises(RuntimeError, match='cannot be differentiated'):
        gh.float().pow(2).sum().backward()


def test_arguments_changed_before_the_backward_pass_are_noticed():
    x, w = _dev(U.normal(1, 8, 64)).requires_grad_(), _dev(U.normal(2, 32, 64)).requires_grad_()
    y = deep_ep.grouped_linear(x, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


# ---- together, as they are used -----------------------------------------------------------------------------

def _moe(tokens, hidden, inner, experts, topk, alignment, seed=0):
    from helpers import make_routing
    idx, weights = make_routing(tokens, experts, topk, seed=seed, masked=0.1)
    x = U.normal(seed, tokens, hidden)
    up, down = U.normal(seed + 1, experts, 2 * inner, hidden, scale=hidden ** -0.5), U.normal(seed + 2, experts, hidden, inner, scale=inner ** -0.5)
    buf = deep_ep.EPBuffer(deep_ep.LocalGroup(), num_max_tokens_per_rank=tokens, hidden=hidden, num_topk=topk)
    return x, idx, weights, up, down, buf


def _moe_values(x, idx, weights, up, down):
    out = torch.zeros(x.shape, dtype=torch.float64)
    for t in range(x.size(0)):
        for k in range(idx.size(1)):
            e = int(idx[t, k])
            if e >= 0:
                h = x[t] @ up[e].t()
                gate, u = h.chunk(2)
                out[t] = out[t] + (gate * torch.sigmoid(gate) * u * weights[t, k]) @ down[e].t()
    return out


@pytest.mark.parametrize('sync', [False, True])
@pytest.mark.parametrize('alignment', [1, 128])
@pytest.mark.parametrize('fp8', [False, True])
def test_dispatch_experts_combine(sync, alignment, fp8):
    tokens, hidden, inner, experts, topk = 77, 256, 128, 9, 3
    x, idx, weights, up, down, buf = _moe(tokens, hidden, inner, experts, topk, alignment)
    recv, _, recv_w, handle, _ = buf.dispatch(_dev(x), topk_idx=_dev(idx), topk_weights=_dev(weights), num_experts=experts,
                                              expert_alignment=alignment, do_expand=True, do_cpu_sync=sync, fused_fp8_quant=fp8)
    wu, wd = (U.quantise_weights(up), U.quantise_weights(down)) if fp8 else (up, down)
    h = deep_ep.grouped_linear(recv, _dev(wu), handle)
    a = deep_ep.swiglu(h, handle, recv_w, fused_fp8_quant=fp8)
    y = deep_ep.grouped_linear(a, _dev(wd), handle)
    out, _, _ = buf.combine(y, handle)
    wx = U.widen_rows(U.quantise_rows(x)) if fp8 else x.double()
    want = _moe_values(wx, idx, weights.double(), U.widen_weights(wu), U.widen_weights(wd))
    # three roundings to BF16 (h, y, out) and one of the activation; in FP8 the activation's is 2^-4 of it; relative to the values' size
    rel = (out.cpu().double() - want).norm() / want.norm()
    assert rel <= (2.0 ** -4 + 4 * U.HALF_BF16 if fp8 else 6 * U.HALF_BF16), rel


def test_training_step_of_the_experts():
    """Forward and backward through dispatch, experts and combine, against the gradients of the formula in 64 bits."""
    tokens, hidden, inner, experts, topk = 40, 128, 64, 5, 2
    x, idx, weights, up, down, buf = _moe(tokens, hidden, inner, experts, topk, 16)
    grad_out = U.normal(7, tokens, hidden)
    rx, rw, ru, rd = (t.double().requires_grad_() for t in (x, weights, up, down))
    _moe_values(rx, idx, rw, ru, rd).backward(grad_out.double())
    with torch.no_grad():
        recv, _, recv_w, handle, _ = buf.dispatch(_dev(x), topk_idx=_dev(idx), topk_weights=_dev(weights), num_experts=experts,
                                                  expert_alignment=16, do_expand=True)
    recv, recv_w = recv.requires_grad_(), recv_w.requires_grad_()
    du, dd = _dev(up).requires_grad_(), _dev(down).requires_grad_()
    y = deep_ep.grouped_linear(deep_ep.swiglu(deep_ep.grouped_linear(recv, du, handle), handle, recv_w), dd, handle)
    out, _, _ = buf.combine(y.detach(), handle)
    grad_rows, _, _, _, _ = buf.dispatch(_dev(grad_out), handle=handle, do_expand=True)
    y.backward(grad_rows)
    grad_x, grad_w, _ = buf.combine(recv.grad, handle, topk_weights=recv_w.grad)
    rel = lambda got, want: ((got.cpu().double() - want).norm() / want.norm()).item()  # noqa: E731
    # at most six roundings to BF16 on the way to each of them
    for got, want in ((grad_x, rx.grad), (grad_w, rw.grad), (du.grad, ru.grad), (dd.grad, rd.grad)):
        assert rel(got, want) <= 8 * U.HALF_BF16


def test_adapters_of_tokens_behind_a_dispatch():
    tokens, hidden, experts, topk, adapters = 50, 128, 6, 2, 4
    x, idx, weights, up, _, buf = _moe(tokens, hidden, 64, experts, topk, 8)
    of_token = torch.randint(-1, adapters, (tokens,), generator=torch.Generator().manual_seed(3)).to(torch.int32)
    a, b = U.normal(4, adapters, experts, 16, hidden, scale=hidden ** -0.5), U.normal(5, adapters, experts, 128, 16)
    for sync in (False, True):
        recv, _, _, handle, _ = buf.dispatch(_dev(x), topk_idx=_dev(idx), topk_weights=_dev(weights), num_experts=experts, expert_alignment=8,
                                             do_expand=True, do_cpu_sync=sync)
        of_row = deep_ep.expand_token_index(handle, _dev(of_token))
        assert of_row.shape == (handle.num_expanded_tokens,)
        slots = handle.recv_src_metadata.cpu()
        want = torch.full((handle.num_expanded_tokens,), -1, dtype=torch.int32)
        for row in slots[:int(handle.psum_num_recv_tokens_per_rank.cpu()[-1])]:
            for s in row[:topk]:
                if s >= 0:
                    want[s] = of_token[row[topk]]
        assert torch.equal(of_row.cpu(), want)
        y = deep_ep.grouped_lora_linear(recv, _dev(up), _dev(a), _dev(b), of_row, handle)
        assert y.shape == (recv.size(0), 128)
    s, e = next((int(r[k]), int(idx[r[topk], k])) for r in slots for k in range(topk) if r[k] >= 0 and of_token[r[topk]] >= 0)
    row, n = recv[s].cpu().double(), int(want[s])
    value = row @ up[e].double().t() + (row @ a[n, e].double().t()) @ b[n, e].double().t()
    assert ((y[s].cpu().double() - value).norm() / value.norm()) <= 2 * U.HALF_BF16


def test_captured_with_a_dispatch_and_replayed():
    """Dispatch, experts with adapters, combine in one graph, replayed over new inputs, with eager work between."""
    tokens, hidden, inner, experts, topk = 32, 256, 128, 8, 2
    x, idx, weights, up, down, buf = _moe(tokens, hidden, inner, experts, topk, 16)
    up, down = _dev(up), _dev(down)
    a, b = _dev(U.normal(4, 3, experts, 8, hidden, scale=hidden ** -0.5)), _dev(U.normal(5, 3, experts, 2 * inner, 8))
    static = [_dev(x), _dev(idx), _dev(weights), _dev(torch.zeros(tokens, dtype=torch.int32))]

    def step():
        recv, _, recv_w, handle, _ = buf.dispatch(static[0], topk_idx=static[1], topk_weights=static[2], num_experts=experts,
                                                  expert_alignment=16, do_expand=True, do_cpu_sync=False)
        of_row = deep_ep.expand_token_index(handle, static[3])
        h = deep_ep.grouped_lora_linear(recv, up, a, b, of_row, handle)
        y = deep_ep.grouped_linear(deep_ep.swiglu(h, handle, recv_w), down, handle)
        gx, gw = deep_ep.grouped_linear_grad(y, deep_ep.swiglu(h, handle, recv_w), down, handle, need_x=False)
        return buf.combine(y, handle)[0], gw

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        nx, nidx, nw, *_ = _moe(tokens, hidden, inner, experts, topk, 16, seed=10 + seed)
        for s, v in zip(static, (nx, nidx, nw, torch.randint(-1, 3, (tokens,), generator=torch.Generator().manual_seed(seed)).to(torch.int32))):
            s.copy_(v)
        graph.replay()
        got = [t.clone() for t in captured]
        for g, w in zip(got, step()):
            assert torch.equal(g, w)
        torch.cuda.synchronize()


def test_results_do_not_lie_on_operands():
    x, w, psum = _dev(U.normal(1, 8, 64)), _dev(U.normal(2, 64, 64)), _dev(torch.tensor([8], dtype=torch.int32))
    a, b, idx = _dev(U.normal(3, 1, 8, 64)), _dev(U.normal(4, 1, 64, 8)), torch.zeros(8, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError):
        deep_ep.grouped_linear(x, w, out=x)
    with pytest.raises(RuntimeError):
        deep_ep.grouped_linear(x, w, out=w[8:16])
    with pytest.raises(RuntimeError):
        deep_ep.grouped_lora_linear(x, w, a, b, idx, out=x)
    with pytest.raises(RuntimeError):
        deep_ep.grouped_linear_grad(w, w, w, need_x=False, grad_weight=w)
    h = _dev(U.normal(5, 64, 64))
    with pytest.raises(RuntimeError):
        deep_ep.swiglu(h, out=h.view(-1)[:64 * 32].view(64, 32))


def test_captured_backward_pass_and_replayed():
    layout = U.Layout([300, 20], 16)
    psum = layout.on(DEV)
    inputs = [_dev(U.normal(1, layout.rows, 256)), _dev(U.normal(2, 2, 256, 256)), torch.rand(layout.rows, device=DEV), _dev(U.normal(3, layout.rows, 128))]

    def step(x, w, g, grad):
        x, w, g = (t.detach().requires_grad_() for t in (x, w, g))
        deep_ep.swiglu(deep_ep.grouped_linear(x, w, psum), psum, g, do_zero_padding=True).backward(grad)
        return x.grad, w.grad, g.grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*inputs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*inputs)
    for seed in range(4):
        inputs[0].copy_(U.normal(10 + seed, layout.rows, 256))
        inputs[3].copy_(U.normal(20 + seed, layout.rows, 128))
        graph.replay()
        got = [t.clone() for t in captured]
        for g, w in zip(got, step(*inputs)):
            assert torch.equal(g, w)
        torch.cuda.synchronize()


@pytest.mark.parametrize('kind', ['linear', 'swiglu'])
def test_captured_backward_pass_beside_an_eager_graph_is_refused(kind):
    x, w = _dev(U.normal(1, 8, 64)).requires_grad_(), _dev(U.normal(2, 64, 64)).requires_grad_()
    run = (lambda: deep_ep.grouped_linear(x, w)) if kind == 'linear' else (lambda: deep_ep.swiglu(x))
    eager = run()
    grad = torch.ones_like(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
        with pytest.raises(RuntimeError, match='while an eager one of the same leaves lives'):
            y.backward(grad)
    graph.replay()
    assert x.grad is None and torch.equal(y.detach(), eager.detach())
    eager.backward(grad)
    if kind == 'linear':
        assert torch.equal(w.grad, deep_ep.grouped_linear_grad(grad, x.detach(), w.detach())[1])
    else:
        assert torch.equal(x.grad, deep_ep.swiglu_grad(grad, x.detach())[0])


def test_on_another_stream():
    layout = U.Layout([300, 20], 16)
    x, w = _dev(U.normal(1, layout.rows, 256)), _dev(U.normal(2, 2, 256, 256))
    want = deep_ep.grouped_linear(x, w, layout.on(DEV), do_zero_padding=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = x.detach().requires_grad_()
        y = deep_ep.grouped_linear(leaf, w, layout.on(DEV), do_zero_padding=True)
        y.backward(y.detach())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y.detach(), want)
    assert torch.equal(leaf.grad, deep_ep.grouped_linear_grad(want, x, w, layout.on(DEV), need_weight=False, do_zero_padding=True)[0])


def test_results_do_not_change_from_run_to_run():
    layout = U.Layout([513, 40, 7], 32)
    x, w, a, b, scales = (_dev(t) for t in _lora_inputs(layout, 6, 16, 2048, 512, False))
    idx = _dev(torch.randint(-1, 6, (layout.rows,), generator=torch.Generator().manual_seed(2)).to(torch.int32))
    grad = _dev(U.normal(8, layout.rows, 512))

    def once():
        y = deep_ep.grouped_lora_linear(x, w, a, b, idx, layout.on(DEV), scales=scales, do_zero_padding=True)
        return (y, *deep_ep.grouped_linear_grad(grad, x, w, layout.on(DEV), do_zero_padding=True))
    first = once()
    for _ in range(3):
        for f, g in zip(first, once()):
            assert torch.equal(f, g)
