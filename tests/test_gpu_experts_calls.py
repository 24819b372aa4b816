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
