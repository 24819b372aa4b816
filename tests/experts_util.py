"""Layouts, inputs and values in 64 bits for the tests of the experts' computation (all data is made on the CPU)."""
import math

import torch

GROUP = 128
HALF_BF16 = 2.0 ** -8         # a rounding to bfloat16 is off by at most this, relative
STEP_F32 = 2.0 ** -23         # two roundings to float32, relative


class Layout:
    """Expert-major rows with padding, and `tail` rows behind the last expert's."""

    def __init__(self, counts, alignment, tail=0):
        self.counts, self.alignment, self.start = list(counts), alignment, []
        at, ends = 0, []
        for c in counts:
            self.start.append(at)
            ends.append(at + c)
            at = -(-(at + c) // alignment) * alignment
        self.aligned, self.rows = at, at + tail
        self.psum = torch.tensor(ends, dtype=torch.int32)
        self.valid = torch.zeros(self.rows, dtype=torch.bool)
        self.expert = torch.zeros(self.rows, dtype=torch.int64)
        for e, (s, c) in enumerate(zip(self.start, counts)):
            self.valid[s:s + c] = True
            self.expert[s:s + c] = e
        self.padding = ~self.valid & (torch.arange(self.rows) < at)      # what do_zero_padding writes

    def on(self, device):
        return self.psum.to(device), self.alignment

    def slices(self):
        return [slice(s, s + c) for s, c in zip(self.start, self.counts)]


def spoil(t, layout):
    """NaN into the rows of no expert: nothing may come of them."""
    t[~layout.valid] = math.nan
    return t


def normal(seed, *shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(torch.bfloat16)


def quantise_rows(x):
    rows, k = x.shape
    groups = torch.nn.functional.pad(x.float(), (0, -k % GROUP)).view(rows, -1, GROUP)
    scale = groups.abs().amax(dim=2).clamp(1e-4) / 448.0
    q = (groups / scale[:, :, None]).to(torch.float8_e4m3fn)
    return q.view(rows, -1)[:, :k].contiguous(), scale


def quantise_weights(w):
    e, n, k = w.shape
    blocks = torch.nn.functional.pad(w.float(), (0, -k % GROUP, 0, -n % GROUP))
    blocks = blocks.view(e, blocks.size(1) // GROUP, GROUP, -1, GROUP)
    scale = blocks.abs().amax(dim=(2, 4)).clamp(1e-4) / 448.0
    q = (blocks / scale[:, :, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(e, blocks.size(1) * GROUP, -1)[:, :n, :k].contiguous(), scale


def widen_rows(x):
    if not isinstance(x, tuple):
        return x.double()
    q, scale = x
    return q.double() * scale.double().repeat_interleave(GROUP, 1)[:, :q.size(1)]


def widen_weights(w):
    if not isinstance(w, tuple):
        return w.double()
    q, scale = w
    scale = scale.double().repeat_interleave(GROUP, 1)[:, :q.size(1)]
    return q.double() * scale.repeat_interleave(GROUP, 2)[:, :, :q.size(2)]


def linear(x, w, layout):
    """(values, sums of the magnitudes of the products) in 64 bits; zeros in rows of no expert."""
    x, w = widen_rows(x), widen_weights(w)
    y = torch.zeros((layout.rows, w.size(1)), dtype=torch.float64)
    size = torch.zeros_like(y)
    for e, mine in enumerate(layout.slices()):
        y[mine] = x[mine] @ w[e].t()
        size[mine] = x[mine].abs() @ w[e].abs().t()
    return y, size


def fp8_error(x, w, layout):
    """What the FP8 matrix instruction leaves out: of eight neighbouring channels' products it keeps what is above 2^-13 of the power of two
    below the largest (truncated; measured with single products, of 1.5 * 2^3 beside 2^15 all, of 1.5 * 2^2 4, of 2 and less nothing).
    Seven of the eight can lose up to that; the largest product of a block is at most the product of the block's largest factors."""
    x, w = widen_rows(x).abs(), widen_weights(w).abs()
    blocks = lambda t: torch.nn.functional.pad(t, (0, -t.size(-1) % 8)).unflatten(-1, (-1, 8)).amax(dim=-1)  # noqa: E731
    x, w = blocks(x), blocks(w)
    error = torch.zeros((layout.rows, w.size(1)), dtype=torch.float64)
    for e, mine in enumerate(layout.slices()):
        error[mine] = x[mine] @ w[e].t() * 7 * 2.0 ** -13
    return error


def weight_grad(grad, x, layout):
    out = torch.zeros((len(layout.counts), grad.size(1), x.size(1)), dtype=torch.float64)
    size = torch.zeros_like(out)
    for e, mine in enumerate(layout.slices()):
        out[e] = grad[mine].double().t() @ x[mine].double()
        size[e] = grad[mine].double().abs().t() @ x[mine].double().abs()
    return out, size


def assert_sum(got, want, size, terms, half=HALF_BF16, what='', more=0.0):
    """`got` is a sum of `terms` products in 32 bits, rounded once: each of the additions (and the scaling of a group) is off by at most a
    step of 2^-23 of the sum of magnitudes, the last rounding by `half` of the value (and of that error).  `more`: what the products lose."""
    got = got.cpu().double()
    assert torch.isfinite(got).all(), what
    error = (terms + 8) * STEP_F32 * size + more
    over = (got - want).abs() - (half * (want.abs() + error) + error + 1e-40)
    worst = over.flatten().argmax() if over.numel() else 0
    assert over.numel() == 0 or over.max() <= 0, f'{what}: {got.flatten()[worst]} for {want.flatten()[worst]}'
