"""Calls of the experts' computation that its documentation allows or refuses: results beside their operands, paths of large calls, counts
that are not the tensors', autograd."""
import pytest
import torch

import deep_ep
import experts_util as U

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def _dev(t):
    return tuple(x.to(DEV) for x in t) if isinstance(t, tuple) else t.to(DEV)


@pytest.mark.parametrize('rows', [20, 700])
def test_results_beside_their_operands(rows):
    """Columns of one matrix are operand and result."""
    x, w = _dev(U.normal(1, rows, 256)), _dev(U.normal(2, 136, 256))
    want = deep_ep.grouped_linear(x, w)
    wide = torch.full((rows, 640), 77.0, dtype=torch.bfloat16, device=DEV)
    vx, out = wide[:, 64:320].copy_(x), wide[:, 320:456]
    assert torch.equal(deep_ep.grouped_linear(vx, w, out=out), want)
    assert torch.equal(vx, x) and (wide[:, :64] == 77).all() and (wide[:, 456:] == 77).all()
    activated = deep_ep.swiglu(x)
    assert torch.equal(deep_ep.swiglu(vx, out=wide[:, 480:608]), activated)
    grad = torch.zeros(rows, 136, dtype=torch.bfloat16, device=DEV).copy_(want)
    _, gw = deep_ep.grouped_linear_grad(grad, x, w, need_x=False)
    ww = torch.zeros(136, 512, dtype=torch.bfloat16, device=DEV)
    vw = ww[:, :256].copy_(w)
    _, vgw = deep_ep.grouped_linear_grad(out, vx, vw, need_x=False, grad_weight=ww[:, 256:])
    assert torch.equal(vgw, gw) and torch.equal(vw, w)


def test_results_on_columns_of_their_operands_are_refused():
    wide, w = torch.zeros(300, 640, dtype=torch.bfloat16, device=DEV), _dev(U.normal(2, 256, 256))
    for at in (0, 8, 248):
        with pytest.raises(deep_ep._C.EPException, match='must not lie on an operand'):
            deep_ep.grouped_linear(wide[:, :256], w, out=wide[:, at:at + 256])
        with pytest.raises(deep_ep._C.EPException, match='must not lie on an operand'):
            deep_ep.swiglu(wide[:, :256], out=wide[:, at:at + 128])
    assert (wide == 0).all()


def test_forward_mode_tangents_of_adapters_are_refused():
    from torch.autograd import forward_ad
    x, w, a, b, scales = (_dev(U.normal(i, *shape)) for i, shape in enumerate([(4, 64), (64, 64), (1, 8, 64), (1, 64, 8), (1,)]))
    idx, scales = torch.zeros(4, dtype=torch.int32, device=DEV), scales.float()
    with forward_ad.dual_level():
        for i in range(3):
            tensors = [a, b, scales]
            tensors[i] = forward_ad.make_dual(tensors[i], torch.ones_like(tensors[i]))
            with pytest.raises(deep_ep._C.EPException, match='forward-mode gradients are not implemented'):
                deep_ep.grouped_lora_linear(x, w, *tensors[:2], idx, scales=tensors[2])


def _stale(saved, store):
    """A graph that saved `saved` notices what `store` wrote into it."""
    w = _dev(U.normal(9, 16, saved.size(1))).requires_grad_()
    y = deep_ep.grouped_linear(saved, w)
    before = saved._version
    store()
    assert saved._version > before
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_stored_results_are_noticed_by_graphs_that_saved_the_tensor():
    x, w, a, b = (_dev(U.normal(i, *shape)) for i, shape in enumerate([(8, 64), (64, 64), (1, 8, 64), (1, 64, 8)]))
    idx, h, grad = torch.zeros(8, dtype=torch.int32, device=DEV), _dev(U.normal(5, 8, 128)), _dev(U.normal(6, 8, 8))
    out = torch.zeros(8, 64, dtype=torch.bfloat16, device=DEV)
    _stale(out, lambda: deep_ep.grouped_linear(x, w, out=out))
    _stale(out, lambda: deep_ep.grouped_lora_linear(x, w, a, b, idx, out=out))
    _stale(out, lambda: deep_ep.swiglu(h, out=out))
    wide = torch.zeros(8, 128, dtype=torch.bfloat16, device=DEV)
    _stale(wide, lambda: deep_ep.grouped_linear(x, w, out=wide[:, 64:]))           # (a view has its base's version)
    _stale(out, lambda: deep_ep.grouped_linear_grad(grad, x, out, need_x=False, grad_weight=out))
    q, sf = torch.zeros(8, 64, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.zeros(8, 1, device=DEV)
    versions = q._version, sf._version
    deep_ep.swiglu(h, fused_fp8_quant=True, out=(q, sf))
    assert q._version > versions[0] and sf._version > versions[1]
    # what only lies beside the result, or is only read, keeps its version
    versions = x._version, w._version, h._version
    deep_ep.swiglu(h, out=deep_ep.grouped_linear(x, w, out=out))
    assert versions == (x._version, w._version, h._version)


def test_results_in_inference_mode():
    x, w = _dev(U.normal(1, 8, 64)), _dev(U.normal(2, 64, 64))
    want = deep_ep.grouped_linear(x, w)
    with torch.inference_mode():
        out = torch.zeros_like(want)
        assert torch.equal(deep_ep.grouped_linear(x, w, out=out), want)
    assert torch.equal(deep_ep.grouped_linear(x, w, out=out), want)      # (such a tensor has no version)


def _captured_while_alive(leaf, run):
    """(the eager result, the error of a captured backward pass beside it, the graph)"""
    eager = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
        with pytest.raises(RuntimeError, match='while an eager one of the same leaves lives'):
            y.backward(torch.ones_like(y))
    graph.replay()
    assert leaf.grad is None and torch.equal(y.detach(), eager.detach())
    eager.backward(torch.ones_like(eager))
    return leaf.grad


def test_leaves_behind_other_nodes_are_seen_when_a_backward_pass_is_captured():
    x, w = _dev(U.normal(1, 8, 64)), _dev(U.normal(2, 64, 64))
    ones = torch.ones(8, 64, dtype=torch.bfloat16, device=DEV)
    gx, gw = deep_ep.grouped_linear_grad(ones, x, w)
    master = w.float().requires_grad_()
    assert torch.equal(_captured_while_alive(master, lambda: deep_ep.grouped_linear(x, master.to(torch.bfloat16))), gw.float())
    rows = x.float().requires_grad_()
    assert torch.equal(_captured_while_alive(rows, lambda: deep_ep.grouped_linear(rows.view(64, 8).view(8, 64).to(torch.bfloat16), w)), gx.float())
    gates = x.float().requires_grad_()
    gh, _ = deep_ep.swiglu_grad(ones[:, :32].contiguous(), x)
    assert torch.equal(_captured_while_alive(gates, lambda: deep_ep.swiglu(gates.to(torch.bfloat16))), gh.float())


def test_leaves_that_a_captured_pass_does_not_go_to_may_be_an_eager_graphs():
    x, w = _dev(U.normal(1, 8, 64)), _dev(U.normal(2, 64, 64)).requires_grad_()
    grad = _dev(U.normal(3, 8, 64))
    eager = deep_ep.grouped_linear(x, w)

    def step():
        leaf = x.detach().requires_grad_()
        y = deep_ep.grouped_linear(leaf, w)
        return torch.autograd.grad(y, leaf, grad)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        x.copy_(U.normal(10 + seed, 8, 64)), grad.copy_(U.normal(20 + seed, 8, 64))
        graph.replay()
        got = captured.clone()
        assert torch.equal(got, deep_ep.grouped_linear_grad(grad, x, w.detach(), need_weight=False)[0])
        torch.cuda.synchronize()
    assert eager.requires_grad


# ---- launches that only some sizes take ---------------------------------------------------------------------

def _lora_inputs(layout, adapters, rank, depth, columns):
    experts = len(layout.counts)
    x, w = U.normal(1, layout.rows, depth), U.normal(2, experts, columns, depth, scale=depth ** -0.5)
    a, b = U.normal(3, adapters, experts, rank, depth, scale=depth ** -0.5), U.normal(4, adapters, experts, columns, rank)
    scales = torch.rand(adapters, generator=torch.Generator().manual_seed(5)) + 0.5
    idx = torch.randint(-1, adapters + 1, (layout.rows,), generator=torch.Generator().manual_seed(6)).to(torch.int32)
    return x, w, a, b, scales, idx


def _lora_values(x, w, a, b, scales, idx, layout):
    """(values, sums of magnitudes of the product's terms and of the adapters') in 64 bits."""
    y, size = U.linear(x, w, layout)
    low = torch.zeros_like(y)
    for e, mine in enumerate(layout.slices()):
        for n in range(a.size(0)):
            rows = torch.arange(layout.rows)[mine][idx[mine] == n]
            s = scales[n].double()
            y[rows] += s * (x[rows].double() @ a[n, e].double().t()) @ b[n, e].double().t()
            low[rows] += s * (x[rows].double().abs() @ a[n, e].double().abs().t()) @ b[n, e].double().abs().t()
    return y, size, low


def _in_parts(layout, depth, columns, adapters):
    lib, c64 = deep_ep._C._lib, deep_ep._C.ctypes.c_int64
    f = lib.ep_grouped_linear_workspace_bytes
    f.restype = c64
    return f(c64(layout.rows), len(layout.counts), layout.alignment, c64(depth), c64(columns), int(adapters)) > 0


def _padding_of(got, layout, zeroed):
    assert (got[(~layout.valid & ~layout.padding if zeroed else ~layout.valid).to(DEV)] == 77).all()
    assert not zeroed or (got[layout.padding.to(DEV)] == 0).all()


@pytest.mark.parametrize('counts,alignment,tail', [([1100], 1, 3), ([600, 0, 700], 16, 0)])
@pytest.mark.parametrize('rank', [8, 24, 64])
def test_many_rows_with_adapters_in_parts_of_the_depth(counts, alignment, tail, rank):
    """More rows than come with the parts in one launch: the low-rank rows have one of their own."""
    depth, columns = 7168, 256
    layout = U.Layout(counts, alignment, tail)
    assert layout.rows > 1024 and _in_parts(layout, depth, columns, True)
    x, w, a, b, scales, idx = _lora_inputs(layout, 5, rank, depth, columns)
    want, size, low = _lora_values(x, w, a, b, scales, idx, layout)
    U.spoil(x, layout)
    idx[~layout.valid] = 0
    more = low * (2.0 ** -17 + (depth + rank + 32) * U.STEP_F32)
    v = layout.valid
    for zeroed in (False, True):
        out = torch.full((layout.rows, columns), 77.0, dtype=torch.bfloat16, device=DEV)
        deep_ep.grouped_lora_linear(*(_dev(t) for t in (x, w, a, b, idx)), layout.on(DEV), scales=_dev(scales), out=out, do_zero_padding=zeroed)
        U.assert_sum(out[v.to(DEV)], want[v], size[v], depth, more=more[v])
        _padding_of(out, layout, zeroed)


@pytest.mark.parametrize('rows,columns', [(1100, 256), (2300, 1024)])
def test_adapters_that_are_far_apart(rows, columns):
    """One buffer of 31 bits does not reach all of them: they are multiplied one by one."""
    layout = U.Layout([rows], 1)
    x, w, a, b, scales, idx = (_dev(t) for t in _lora_inputs(layout, 3, 16, 512, columns))
    want = deep_ep.grouped_lora_linear(x, w[0], a[:, 0], b[:, 0], idx, scales=scales)
    far = (1 << 30) + 64
    buffer = torch.empty(2 * far + 16 * 512, dtype=torch.bfloat16, device=DEV)
    wide = buffer.as_strided((3, 16, 512), (far, 512, 1)).copy_(a[:, 0])
    assert torch.equal(deep_ep.grouped_lora_linear(x, w[0], wide, b[:, 0], idx, scales=scales), want)


@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'lora'])
def test_counts_beyond_the_tensors_with_the_depth_in_parts(kind):
    depth, columns, rows = 7168, 256, 40
    x, w = U.normal(1, rows, depth), U.normal(2, 3, columns, depth, scale=depth ** -0.5)
    a, b = _dev(U.normal(3, 2, 3, 16, depth, scale=depth ** -0.5)), _dev(U.normal(4, 2, 3, columns, 16))
    idx = (torch.arange(rows, dtype=torch.int32) % 3 - 1).to(DEV)
    assert _in_parts(U.Layout([30, 8, 0], 16, 0), depth, columns, kind == 'lora')
    x, w = (_dev(U.quantise_rows(x)), _dev(U.quantise_weights(w))) if kind == 'fp8' else (_dev(x), _dev(w))

    def run(psum, out):
        layout = torch.tensor(psum, dtype=torch.int32, device=DEV), 16
        if kind == 'lora':
            return deep_ep.grouped_lora_linear(x, w, a, b, idx, layout, out=out, do_zero_padding=True)
        return deep_ep.grouped_linear(x, w, layout, out=out, do_zero_padding=True)
    wide = torch.full((rows + 64, columns), 77.0, dtype=torch.bfloat16, device=DEV)
    want = run([30, 40, 40], torch.full((rows, columns), 77.0, dtype=torch.bfloat16, device=DEV))
    assert torch.equal(run([30, 200, 2 ** 31 - 1], wide[32:72]), want)
    assert (wide[:32] == 77).all() and (wide[72:] == 77).all()
    wide[32:72] = 77
    want = run([0, 0, 7], torch.full((rows, columns), 77.0, dtype=torch.bfloat16, device=DEV))
    assert torch.equal(run([-5, -(2 ** 31), 7], wide[32:72]), want) and (want[16:] == 77).all()
    run([35, 10, 2 ** 31 - 1], wide[32:72])                        # (in no order: what comes out is not said, where it goes is)
    assert (wide[:32] == 77).all() and (wide[72:] == 77).all()


@pytest.mark.parametrize('rows,in_parts', [(3000, False), (4500, True)])
def test_weight_gradients_of_counts_beyond_the_tensors(rows, in_parts):
    grad, x = _dev(U.normal(1, rows, 72)), _dev(U.normal(2, rows, 136))
    lib, c64 = deep_ep._C._lib, deep_ep._C.ctypes.c_int64
    lib.ep_grouped_weight_grad_workspace_bytes.restype = c64
    assert (lib.ep_grouped_weight_grad_workspace_bytes(c64(rows), 3, 8, c64(72), c64(136)) > 0) == in_parts
    wide = torch.full((5, 72, 136), 77.0, device=DEV)
    w = torch.zeros(3, 72, 136, dtype=torch.bfloat16, device=DEV)

    def run(psum, out):
        return deep_ep.grouped_linear_grad(grad, x, w, (torch.tensor(psum, dtype=torch.int32, device=DEV), 8), need_x=False, grad_weight=out)[1]
    for psum, same in (([1300, 5000, 2 ** 31 - 1], [1300, rows, rows]), ([-7, -(2 ** 31), 2000], [0, 0, 2000])):
        want = run(same, torch.zeros(3, 72, 136, device=DEV))
        assert torch.equal(run(psum, wide[1:4]), want)
        assert (wide[0] == 77).all() and (wide[4] == 77).all()


@pytest.mark.parametrize('fp8', [False, True])
def test_swiglu_of_counts_beyond_the_tensors(fp8):
    h, grad, weights = _dev(U.normal(1, 40, 512)), _dev(U.normal(2, 40, 256)), torch.rand(40, device=DEV)

    def run(psum):
        layout = torch.tensor(psum, dtype=torch.int32, device=DEV), 16
        if fp8:
            q, sf = deep_ep.swiglu(h, layout, weights, fused_fp8_quant=True, do_zero_padding=True)
            return q.view(torch.uint8), sf
        return deep_ep.swiglu(h, layout, weights, do_zero_padding=True), *deep_ep.swiglu_grad(grad, h, layout, weights, do_zero_padding=True)
    for psum, same, rows in (([30, 200, 2 ** 31 - 1], [30, 40, 40], 40), ([-5, -(2 ** 31), 7], [0, 0, 7], 16)):
        for got, want in zip(run(psum), run(same)):
            assert torch.equal(got[:rows], want[:rows])


# ---- several partitions ---------------------------------------------------------------------------------------

@pytest.mark.parametrize('R,max_tokens,E,K,A', [(2, 40, 6, 2, 8), (3, 70, 12, 5, 16), (4, 33, 8, 3, 1)])
@pytest.mark.parametrize('sync', [False, True])
def test_experts_of_several_partitions(R, max_tokens, E, K, A, sync):
    """Tokens of every partition through the experts of each, with the tokens' adapters, and back."""
    from helpers import make_routing
    from test_gpu_node import combine_all, dispatch_all, make_node
    H, N, adapters, epr = 256, 256, 3, E // R
    bufs = make_node(R, max_tokens, H, K, False)
    tokens = [max_tokens - 5 * r for r in range(R)]
    xs = [U.normal(10 + r, t, H) for r, t in enumerate(tokens)]
    routing = [make_routing(t, E, K, seed=20 + r, masked=0.1) for r, t in enumerate(tokens)]
    w = U.normal(1, E, N, H, scale=H ** -0.5)
    a, b = U.normal(2, adapters, E, 16, H, scale=H ** -0.5), U.normal(3, adapters, E, N, 16, scale=0.25)
    of_token = torch.full((R * max_tokens,), 99, dtype=torch.int32)                # (beyond a partition's tokens: nobody's)
    for r, t in enumerate(tokens):
        of_token[r * max_tokens:r * max_tokens + t] = torch.randint(-1, adapters, (t,), generator=torch.Generator().manual_seed(30 + r))
    outs = dispatch_all(bufs, [_dev(x) for x in xs], [_dev(i) for i, _ in routing], [_dev(g) for _, g in routing], num_experts=E,
                        num_max_tokens_per_rank=max_tokens, expert_alignment=A, do_expand=True, do_cpu_sync=sync)
    ys, handles, gates = [], [], []
    for p, (recv, _, recv_w, handle) in enumerate(outs):
        of_row = deep_ep.expand_token_index(handle, _dev(of_token))
        metadata, ranks = handle.recv_src_metadata.cpu(), handle.psum_num_recv_tokens_per_rank.cpu()
        want = torch.full((handle.num_expanded_tokens,), -1, dtype=torch.int32)
        for row in metadata[:int(ranks[-1])].tolist():
            for s in row[:K]:
                if s >= 0:
                    want[s] = of_token[row[K]]
        assert torch.equal(of_row.cpu(), want) and (want < 99).all()
        local = slice(p * epr, (p + 1) * epr)
        ys.append(deep_ep.grouped_lora_linear(recv, _dev(w[local].contiguous()), _dev(a[:, local].contiguous()), _dev(b[:, local].contiguous()), of_row,
                                              handle))
        handles.append(handle), gates.append(recv_w)
    combined = combine_all(bufs, ys, handles, gates, [None] * R)
    for r, t in enumerate(tokens):
        idx, x, want = routing[r][0], xs[r].double(), torch.zeros(t, N, dtype=torch.float64)
        for i in range(t):
            n = int(of_token[r * max_tokens + i])
            for e in idx[i].tolist():
                if e >= 0:
                    want[i] += x[i] @ w[e].double().t()
                    if n >= 0:
                        want[i] += (x[i] @ a[n, e].double().t()) @ b[n, e].double().t()
        got = combined[r][0].cpu().double()
        # one rounding of every expert's row and up to two of their sums
        assert (got - want).norm() <= 3 * U.HALF_BF16 * want.norm()
    for buf in bufs:
        buf.destroy()


# ---- rows and experts that are not finite ----------------------------------------------------------------------

@pytest.mark.parametrize('counts', [[20, 3, 9], [300, 70, 513]])
@pytest.mark.parametrize('depth', [256, 7168])
@pytest.mark.parametrize('kind', ['bf16', 'fp8', 'lora', 'rows'])
@pytest.mark.parametrize('value', [float('inf'), float('nan')])
def test_what_is_not_finite_stays_with_its_row_and_expert(counts, depth, kind, value):
    """A row's values do not reach another row, an expert's weights no other expert's rows: to the last bit what comes without them."""
    layout = U.Layout(counts, 8)
    x, w = U.normal(1, layout.rows, depth), U.normal(2, 3, 256, depth, scale=depth ** -0.5)
    a, b = _dev(U.normal(3, 4, 3, 16, depth, scale=depth ** -0.5)), _dev(U.normal(4, 4, 3, 256, 16))
    # (one adapter a tile, or none: rows beside one that is not finite are summed in the same order)
    idx = torch.zeros(layout.rows, dtype=torch.int32, device=DEV)
    psum = layout.on(DEV)

    def run(x, w):
        if kind == 'lora':
            return deep_ep.grouped_lora_linear(_dev(x), _dev(w), a, b, idx, psum, do_zero_padding=True)
        if kind == 'rows':
            return deep_ep.grouped_linear_grad(_dev(x), _dev(x), _dev(w.transpose(1, 2).contiguous()), psum, need_weight=False, do_zero_padding=True)[0]
        if kind == 'fp8':
            q, sf = U.quantise_rows(torch.nan_to_num(x, 1.0, 1.0, 1.0))
            sf[~torch.isfinite(x).all(dim=1)] = value
            wq, wsf = U.quantise_weights(torch.nan_to_num(w, 1.0, 1.0, 1.0))
            wsf[~torch.isfinite(w).all(dim=2).all(dim=1)] = value
            return deep_ep.grouped_linear((_dev(q), _dev(sf)), (_dev(wq), _dev(wsf)), psum, do_zero_padding=True)
        return deep_ep.grouped_linear(_dev(x), _dev(w), psum, do_zero_padding=True)
    want = run(x, w)
    bad = x.clone()
    mine = torch.zeros(layout.rows, dtype=torch.bool)
    for row in (0, layout.start[2] + counts[2] - 1):
        bad[row, 5], mine[row] = value, True
    got = run(bad, w)
    assert not torch.isfinite(got[mine.to(DEV)]).any()
    if kind == 'lora':      # (beside it, rows may take their low-rank rows in 32 bits instead of two BF16)
        error = (got.double() - want.double())[~mine.to(DEV)].abs()
        low = (_dev(x).double().abs() @ a[0].double().abs().amax(dim=0).t()) @ b[0].double().abs().amax(dim=0).t()
        assert (error <= want[~mine.to(DEV)].double().abs() * 2 * U.HALF_BF16 + 2 * low[~mine.to(DEV)] * (2.0 ** -17 + depth * U.STEP_F32)).all()
    else:
        assert torch.equal(got[~mine.to(DEV)], want[~mine.to(DEV)])
    bad, mine = w.clone(), torch.zeros(layout.rows, dtype=torch.bool)
    bad[1, :, 5], mine[layout.slices()[1]] = value, True
    got = run(x, bad)
    assert not torch.isfinite(got[mine.to(DEV)]).any() and torch.equal(got[~mine.to(DEV)], want[~mine.to(DEV)])


@pytest.mark.parametrize('value', [float('inf'), float('nan')])
def test_gradients_of_what_is_not_finite_stay_with_their_expert(value):
    layout = U.Layout([70, 40, 300], 8)
    grad, x, w = U.normal(1, layout.rows, 136), U.normal(2, layout.rows, 264), _dev(U.normal(3, 3, 136, 264))
    want = deep_ep.grouped_linear_grad(_dev(grad), _dev(x), w, layout.on(DEV), need_x=False)[1]
    grad[layout.start[1] + 39, 7] = value
    got = deep_ep.grouped_linear_grad(_dev(grad), _dev(x), w, layout.on(DEV), need_x=False)[1]
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert not torch.isfinite(got[1, 7]).any()
    rest = torch.arange(136) != 7
    assert torch.equal(got[1, rest.to(DEV)], want[1, rest.to(DEV)])
