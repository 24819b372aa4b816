"""The experts' computation between `EPBuffer.dispatch` and `EPBuffer.combine`, on the rows as the dispatch hands them out:

    recv_x, _, recv_w, handle, _ = buf.dispatch(x, topk_idx=idx, topk_weights=w, num_experts=E, do_expand=True)
    h = grouped_linear(recv_x, w_gate_up, handle)           # [rows, 2 * I]: gates, then ups
    a = swiglu(h, handle, recv_w)                           # [rows, I], times the rows' gate weights
    y = grouped_linear(a, w_down, handle)
    out, _, _ = buf.combine(y, handle)

The reference leaves the experts to its callers; these are entry points of this library.  All of them

* take the layout as the `EPHandle` of the dispatch, as a pair `(psum_num_recv_tokens_per_expert, expert_alignment)`, or None where one
  matrix serves all rows;
* read the experts' counts on the device: nothing waits for the host, so they may follow a dispatch without a host sync, and be
  recorded into a HIP graph together with it;
* work on tensors of the dispatch's worst-case size as on exact ones.  Rows of no expert (alignment padding and whatever lies behind the
  last expert's rows) are read for nothing.  They stay as they were in `out` and undefined in a result that is allocated here, but that
  `do_zero_padding` writes zeros into the padding rows, as a dispatch does;
* are enqueued on the current stream, on the device of their tensors, which has to be the current one;
* hold sums in 32 bits and round once; nothing is added atomically, results are the same from call to call.  Two places keep less: of eight
  neighbouring channels' products of FP8 the matrix instruction leaves out what is below 2^-13 of the largest (about 3e-5 of a result, beside
  the 2^-8 of its rounding), and `grouped_lora_linear` may keep 2^-17 of a low-rank row;
* refuse tensors with a forward-mode tangent.

A backward pass can be recorded into a HIP graph too, but not while an eager graph of the same leaves lives (RuntimeError): end that one first, or
record `grouped_linear_grad` and `swiglu_grad`.  `out` must not lie on an operand (an error; disjoint columns of one matrix may be both),
nor ask for a gradient itself.

Rows may have any stride that keeps them on 16 bytes; channels are contiguous, and come in multiples of 8 (16 for FP8).
"""
from typing import Optional, Tuple, Union

import torch

from . import _C
from .buffers.ep import EPHandle

_native = _C._native
_Layout = Union[EPHandle, Tuple[torch.Tensor, int], None]
_TensorOrPair = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def _layout(layout: _Layout) -> Tuple[Optional[torch.Tensor], int]:
    if layout is None:
        return None, 1
    if isinstance(layout, EPHandle):
        return layout.psum_num_recv_tokens_per_expert, layout.expert_alignment
    psum, alignment = layout
    return psum, alignment


def _pair(x: _TensorOrPair) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    return x if isinstance(x, tuple) else (x, None)


def _wants_grad(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def grouped_linear(x: _TensorOrPair, weight: _TensorOrPair, layout: _Layout = None, *, out: Optional[torch.Tensor] = None,
                   do_zero_padding: bool = False) -> torch.Tensor:
    """Every expert's rows times that expert's weights: `y[m] = weight[e(m)] @ x[m]`.

    Arguments:
        x: `[rows, K]` bfloat16, or the pair `(float8_e4m3fn [rows, K], float32 [rows, ceil(K / 128)])` that a dispatch with
            `fused_fp8_quant` or `swiglu` with it returns (scales of any strides).
        weight: `[experts, N, K]` bfloat16, or a pair of float8_e4m3fn weights and float32 scales of blocks of 128 x 128,
            `[experts, ceil(N / 128), ceil(K / 128)]`; without the experts' dimension where `layout` is None.
        layout: see the module.
        out: `[rows, N]` bfloat16 to store into.
        do_zero_padding: write zeros into the padding rows.

    Returns `[rows, N]` bfloat16.  Differentiable in `x` and `weight` for bfloat16 without `out`; the gradient of rows of no expert
    is zero, whatever the result's gradient holds there.
    """
    (x, x_sf), (weight, weight_sf), (psum, alignment) = _pair(x), _pair(weight), _layout(layout)
    if _wants_grad(x, weight, x_sf, weight_sf, out):
        if out is not None or x_sf is not None or weight_sf is not None:
            raise AssertionError('gradients are implemented for bfloat16 and without `out`')
        return _native.grouped_linear_autograd(x, weight, psum, alignment, do_zero_padding)
    return _native.grouped_linear(x, x_sf, weight, weight_sf, psum, alignment, out, do_zero_padding, False)


def grouped_linear_grad(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, layout: _Layout = None, *, need_x: bool = True,
                        need_weight: bool = True, grad_weight: Optional[torch.Tensor] = None, accumulate: bool = False,
                        do_zero_padding: bool = False) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients of `grouped_linear` without autograd: `(grad_x [rows, K], grad_weight` like `weight)`, bfloat16.

    Arguments:
        grad: `[rows, N]` bfloat16, gradient of the result.
        need_x, need_weight: what to compute; None in the place of the other.
        grad_weight: a tensor like `weight`, bfloat16 or float32, to store the weights' gradient into.
        accumulate: add to what `grad_weight` (float32) holds instead.
    """
    psum, alignment = _layout(layout)
    grad = _native.rows_of(grad)
    grad_x = _native.grouped_linear(grad, None, weight, None, psum, alignment, None, do_zero_padding, True) if need_x else None
    if not need_weight:
        return grad_x, None
    if grad_weight is None:
        assert not accumulate, 'accumulate=True adds to `grad_weight`'
        grad_weight = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device)
    assert grad_weight.shape == weight.shape
    if _wants_grad(grad_weight):
        raise AssertionError('gradients are stored into tensors without a gradient of their own')
    return grad_x, _native.grouped_weight_grad(grad, x, psum, weight.size(0) if weight.dim() == 3 else 1, alignment, grad_weight, accumulate)


def _num_experts(psum: Optional[torch.Tensor]) -> int:
    return 1 if psum is None else psum.size(0)


def swiglu(h: torch.Tensor, layout: _Layout = None, topk_weights: Optional[torch.Tensor] = None, *, fused_fp8_quant: bool = False,
           out: Optional[_TensorOrPair] = None, do_zero_padding: bool = False) -> _TensorOrPair:
    """The gated activation between an expert's two products: `silu(h[:, :I]) * h[:, I:]`, times the row's gate weight.

    Arguments:
        h: `[rows, 2 * I]` bfloat16: gates, then ups.
        topk_weights: `[rows]` float32, as a dispatch hands them out (`recv_topk_weights`), or None.
        fused_fp8_quant: return `(float8_e4m3fn [rows, I], float32 [rows, ceil(I / 128)])`, quantised as
            `per_token_cast_to_fp8` does (from the values in 32 bits), for the next product.
        out: `[rows, I]` bfloat16, or with `fused_fp8_quant` the pair, to store into.
        do_zero_padding: write zeros into the padding rows (their scales too).

    Differentiable in `h` and `topk_weights` without `fused_fp8_quant` and `out`.
    """
    psum, alignment = _layout(layout)
    out, out_sf = _pair(out)
    assert out is None or (out_sf is not None) == fused_fp8_quant, 'a pair of tensors is what a quantised result is stored into'
    if _wants_grad(h, topk_weights, out, out_sf):
        if out is not None or fused_fp8_quant:
            raise AssertionError('gradients are implemented for bfloat16 and without `out`')
        return _native.swiglu_autograd(h, topk_weights, psum, _num_experts(psum), alignment, do_zero_padding)
    result, sf = _native.swiglu(h, topk_weights, psum, _num_experts(psum), alignment, fused_fp8_quant, out, out_sf, do_zero_padding)
    return (result, sf) if fused_fp8_quant else result


def swiglu_grad(grad: torch.Tensor, h: torch.Tensor, layout: _Layout = None, topk_weights: Optional[torch.Tensor] = None, *,
                do_zero_padding: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of `swiglu` without autograd: `(grad_h [rows, 2 * I] bfloat16, grad_topk_weights [rows] float32` or None `)`."""
    psum, alignment = _layout(layout)
    return _native.swiglu_grad(_native.rows_of(grad), h, topk_weights, psum, _num_experts(psum), alignment, do_zero_padding)


def grouped_lora_linear(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter_idx: torch.Tensor,
                        layout: _Layout = None, *, scales: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                        do_zero_padding: bool = False) -> torch.Tensor:
    """`grouped_linear` with low-rank adapters of many requests beside the experts' weights, or (without a layout) beside one
    projection that all rows share: `y[m] = weight[e] @ x[m] + scales[a] * lora_b[a, e] @ (lora_a[a, e] @ x[m])` with the row's expert
    `e` and adapter `a = adapter_idx[m]`.

    Arguments:
        x: `[rows, K]` bfloat16; weight: `[experts, N, K]` or `[N, K]` bfloat16.
        lora_a: `[adapters, experts, R, K]` bfloat16, lora_b: `[adapters, experts, N, R]`; without the experts' dimension where there is one.
            R is a multiple of 8 up to 64.
        adapter_idx: `[rows]` int32; a row whose number is outside `[0, adapters)` has no adapter.  `expand_token_index` makes it from
            the tokens' numbers.  An adapter with infinities or NaN changes the rows that have it, no others.
        scales: `[adapters]` float32 or None.
        layout, out, do_zero_padding: as for `grouped_linear`.

    The low-rank rows are sums in 32 bits.  Where a tile of rows has few adapters they go on as two bfloat16 (2^-17 of them is kept), elsewhere in
    32 bits: a row's last bits can depend on the other rows of the call.  For inference: no gradients.
    """
    psum, alignment = _layout(layout)
    if _wants_grad(x, weight, lora_a, lora_b, scales, out):
        raise AssertionError('gradients of adapters are not implemented')
    return _native.grouped_lora_linear(x, weight, lora_a, lora_b, adapter_idx, scales, psum, alignment, out, do_zero_padding)


def expand_token_index(handle: EPHandle, values: torch.Tensor) -> torch.Tensor:
    """A number of every token, such as its adapter's, at the rows that the dispatch made of it: `[num_expanded_tokens]` int32, -1 in
    rows of no expert.  `values`: `[num_tokens]` int32; of several partitions all tokens', partition p's from
    `p * num_max_tokens_per_rank` on."""
    if handle.recv_src_metadata is None:
        raise AssertionError('the handle comes from a dispatch that ran its epilogue')
    return _native.expand_token_index(values, handle.recv_src_metadata, handle.psum_num_recv_tokens_per_rank, handle.num_expanded_tokens)
