"""Times of the operators between a dispatch and a combine: what a program does with the rows that `EPBuffer.dispatch` hands out before
it gives them to `EPBuffer.combine`.

A case is a dict of plain values.  Five kinds:

  linear        the product of every expert's rows with that expert's weights, `deep_ep.grouped_linear`; `payload` 'bf16', or 'fp8'
                with one scale a row and 128 channels and one a 128 x 128 block of the weights
  linear_train  the same in bfloat16 with the gradients of rows and weights
  swiglu        silu(gate) * up * the row's gate weight, `deep_ep.swiglu`; `payload` 'fp8' quantises the result for the next product
  swiglu_train  the same in bfloat16 with the gradients of rows and gate weights
  lora          `deep_ep.grouped_lora_linear`: products with low-rank adapters of many requests beside the experts' weights; with
                `experts` 0 beside one projection that all rows share

`rows` counts the selected (token, expert) pairs, `k` and `n` are the channels of a row before and after; `zipf` 0 means near-uniform
popularity of the experts, `alignment` is the dispatch's.  `bound`: the tensors have the dispatch's worst-case number of rows, as without
a host sync, and the result is stored into a tensor of the caller's, whose other rows stay as they were.  Where it is false the tensors
have exactly the aligned rows, and padding rows of the result are asked for as zeros.  How many rows the experts have is the case's,
which expert has how many is the seed's.
"""
import math
import os
import sys
import zlib

import numpy as np
import torch

own = False

DEVICE = 'cuda'
GROUP = 128            # channels that share a scale
FP8_MAX = 448.0


def _case(kind, name=None, **values):
    case = dict(kind=kind, rows=0, experts=8, alignment=128, zipf=0.0, bound=False, payload='bf16', k=0, n=0, adapters=0, rank=0,
                requests=0)
    case.update(values)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # the smallest layer that the tests know: 128 tokens of 256 channels, top-2 of 8 experts
        _case('linear', 'toy_bf16', rows=256, alignment=1, k=256, n=512),
        # decode of single tokens: 61 tokens, top-6 of 160 experts, most of which have no row, one or a few
        _case('linear', 'decode_bf16', rows=366, experts=160, alignment=1, bound=True, k=5120, n=2048),
        # decode on one GPU's share of an expert-parallel group: 32 experts, hot and empty ones
        _case('linear', 'decode_fp8', rows=1024, experts=32, alignment=16, zipf=1.2, bound=True, payload='fp8', k=7168, n=4096),
        # the projection back to the hidden size in a prefill
        _case('linear', 'prefill_down_bf16', rows=65536, experts=32, k=2048, n=7168),
        # gate and up projection of the prefill that the framework's benchmark quotes (16384 tokens, top-6)
        _case('linear', 'prefill_up_fp8', rows=98304, experts=64, payload='fp8', k=7168, n=4096),
        # a small fine-tuning step, odd counts, hot and empty experts
        _case('linear_train', 'train_ragged', rows=7147, experts=64, alignment=32, zipf=0.6, k=2560, n=1536),
        # a training step's experts: 8192 tokens, top-4
        _case('linear_train', 'train', rows=32768, experts=16, alignment=64, k=4096, n=2048),
        # between the two products of a decode step
        _case('swiglu', 'decode_swiglu_fp8', rows=1024, experts=32, alignment=16, zipf=1.2, bound=True, payload='fp8', n=2048),
        # between the two products of the benchmark's prefill
        _case('swiglu', 'prefill_swiglu_fp8', rows=98304, experts=64, payload='fp8', n=2048),
        # ... and of a training step
        _case('swiglu_train', 'train_swiglu', rows=32768, experts=16, alignment=64, n=1024),
        # single tokens of 61 requests with adapters of their own beside a projection that all share
        _case('lora', 'decode_lora_shared', rows=61, experts=0, alignment=1, k=7168, n=4096, adapters=32, rank=16, requests=61),
        # a prefill chunk of a few requests, adapters on every expert
        _case('lora', 'prefill_lora', rows=16384, experts=8, k=4096, n=2048, adapters=8, rank=32, requests=12),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(work(c)['flops'] for c in listed())
    while True:
        kind = rng.choice(['linear', 'linear', 'linear_train', 'swiglu', 'swiglu_train', 'lora'])
        wide = kind.startswith('swiglu')
        values = dict(rows=_log_uniform(rng, 1, 98304 if kind in ('linear', 'swiglu') else 32768),
                      experts=rng.choice([1, 3, 8, 8, 16, 32, 64, 160]), alignment=rng.choice([1, 16, 32, 64, 128, 128]),
                      zipf=rng.choice([0.0, 0.0, 0.6, 1.2]), payload=rng.choice(['bf16', 'fp8']) if kind in ('linear', 'swiglu') else 'bf16',
                      k=0 if wide else rng.choice([256, 2048, 2560, 4096, 5120, 7168, 16 * rng.randint(16, 448)]),
                      n=rng.choice([512, 1024, 2048, 2560, 8 * rng.randint(32, 512), 16 * rng.randint(16, 256)]))
        values['bound'] = kind in ('linear', 'swiglu', 'lora') and values['rows'] <= 2048 and rng.random() < 0.5
        if kind == 'lora':
            if rng.random() < 0.4:
                values.update(experts=0, alignment=1, zipf=0.0, bound=False)
            values.update(adapters=rng.choice([1, 2, 5, 8, 16, 32]), rank=rng.choice([8, 16, 16, 32, 64]))
            values['requests'] = min(values['rows'], _log_uniform(rng, 1, 128))
        case = _case(kind, **values)
        experts = max(1, case['experts'])
        weights = experts * case['k'] * case['n']
        # padded copies of the plain form: every expert as long as the longest
        padded = experts * int(_counts(case).max()) * (case['k'] + case['n'])
        adapters = experts * case['adapters'] * case['rank'] * (case['k'] + case['n'])
        if work(case)['flops'] <= most / (3 if kind != 'linear' else 1) and weights <= 2 ** 31 and padded <= 2 ** 31 and adapters <= 2 ** 29:
            return case


# ---- the layout ---------------------------------------------------------------------------------------

def _counts(case):
    """Rows of each expert; the same for every seed but for their order."""
    experts = max(1, case['experts'])
    rng = np.random.RandomState(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != 'name')).encode()) & 0x7fffffff)
    p = np.arange(1, experts + 1, dtype=np.float64) ** -case['zipf']
    return rng.multinomial(case['rows'], p / p.sum())


def _num_rows(case, counts):
    a = case['alignment']
    if case['bound']:
        return -(-(case['rows'] + (a - 1) * len(counts)) // a) * a
    return int(((counts + a - 1) // a * a).sum())


def _layout(case, seed):
    """Counts in this seed's order, first rows of the experts, the handle's prefix sums, the number of rows in all."""
    counts = np.random.RandomState(seed & 0x7fffffff).permutation(_counts(case))
    a = case['alignment']
    aligned = (counts + a - 1) // a * a
    start = np.concatenate([[0], np.cumsum(aligned)[:-1]]) if len(counts) else np.zeros(0)
    return counts, start.astype(np.int64), (start + counts).astype(np.int32), _num_rows(case, counts)


def _valid(counts, start, rows):
    valid = np.zeros(rows, dtype=bool)
    for c, s in zip(counts, start):
        valid[s:s + c] = True
    return torch.from_numpy(valid).to(DEVICE)


# ---- inputs -------------------------------------------------------------------------------------------

def _normal(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)


def _rows_of_tokens(gen, rows, channels):
    """Normal values with one outlier in a thousand."""
    x = _normal(gen, rows, channels)
    outlier = torch.rand((rows, channels), generator=gen, device=DEVICE, dtype=torch.float32) < 1e-3
    return torch.where(outlier, x * 20, x)


def _quantise_rows(x):
    rows, channels = x.shape
    groups = torch.nn.functional.pad(x, (0, -channels % GROUP)).float().view(rows, -1, GROUP)
    scale = groups.abs().amax(dim=2).clamp(1e-4) / FP8_MAX
    q = (groups / scale[:, :, None]).to(torch.float8_e4m3fn)
    return q.view(rows, -1)[:, :channels].contiguous(), scale


def _quantise_weights(w):
    n, k = w.shape
    blocks = torch.nn.functional.pad(w, (0, -k % GROUP, 0, -n % GROUP)).float()
    blocks = blocks.view(blocks.size(0) // GROUP, GROUP, -1, GROUP)
    scale = blocks.abs().amax(dim=(1, 3)).clamp(1e-4) / FP8_MAX
    q = (blocks / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(blocks.size(0) * GROUP, -1)[:n, :k].contiguous(), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, k, n = case['kind'], case['k'], case['n']
    counts, start, ends, rows = _layout(case, seed)
    experts, fp8 = len(counts), case['payload'] == 'fp8'
    state = {'case': case, 'alignment': case['alignment'], 'psum': torch.from_numpy(ends).to(DEVICE)}

    # what the plain form needs of the layout: the place of every row among its expert's, and the rows of every expert
    position = np.zeros((2, rows), dtype=np.int64)
    for e, (c, s) in enumerate(zip(counts, start)):
        position[0, s:s + c] = e
        position[1, s:s + c] = np.arange(c)
    longest = max(1, int(counts.max()))
    table = np.minimum(start[:, None] + np.arange(longest)[None, :], max(0, rows - 1))
    state['expert'], state['place'] = torch.from_numpy(position).to(DEVICE)
    state['table'] = torch.from_numpy(table).to(DEVICE)
    state['filled'] = torch.from_numpy(np.arange(longest)[None, :] < counts[:, None]).to(DEVICE)
    state['valid'] = valid = _valid(counts, start, rows)

    if kind.startswith('swiglu'):
        state['h'] = (_normal(gen, rows, 2 * n) * 1.5) * valid[:, None]
        state['weights'] = torch.rand((rows,), generator=gen, device=DEVICE) * valid
        if kind == 'swiglu_train':
            state['grad'] = _normal(gen, rows, n) * valid[:, None]
        elif case['bound']:
            state['out'] = (torch.zeros((rows, n), device=DEVICE, dtype=torch.uint8).view(torch.float8_e4m3fn),
                            torch.zeros((rows, -(-n // GROUP)), device=DEVICE)) if fp8 else \
                torch.zeros((rows, n), device=DEVICE, dtype=torch.bfloat16)
        return state

    x = _rows_of_tokens(gen, rows, k) * valid[:, None]
    scale = 1 / math.sqrt(k)
    if fp8:
        state['x'] = _quantise_rows(x)
        parts = [_quantise_weights(_normal(gen, n, k) * scale) for _ in range(experts)]
        state['w'] = tuple(torch.stack(p) for p in zip(*parts))
    else:
        state['x'] = x
        w = _normal(gen, experts, n, k).mul_(scale)
        state['w'] = w if case['experts'] else w[0]
    if kind == 'linear_train':
        state['grad'] = _normal(gen, rows, n) * valid[:, None]
    if case['bound']:
        state['out'] = torch.zeros((rows, n), device=DEVICE, dtype=torch.bfloat16)
    if kind == 'lora':
        shared = () if case['experts'] == 0 else (experts,)
        state['a'] = _normal(gen, case['adapters'], *shared, case['rank'], k).mul_(scale)
        state['b'] = _normal(gen, case['adapters'], *shared, n, case['rank']).mul_(1 / math.sqrt(case['rank']))
        state['scales'] = torch.rand((case['adapters'],), generator=gen, device=DEVICE) + 0.5
        # the requests' tokens come one after the other in every expert's rows; one request in eight has no adapter
        request = np.random.RandomState((seed + 1) & 0x7fffffff).randint(0, case['adapters'] + -(-case['adapters'] // 8), case['requests'])
        request[request >= case['adapters']] = -1
        adapter = np.full(rows, -1, dtype=np.int32)
        for c, s in zip(counts, start):
            adapter[s:s + c] = request[np.arange(c) * case['requests'] // max(1, c)]
        state['adapter'] = torch.from_numpy(adapter).to(DEVICE)
    return state


# ---- one pass -----------------------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    sys.path[:0] = [p for p in (os.path.join(os.getcwd(), 'deepep-ascend_amd'),) if p not in sys.path]
    import deep_ep
    case = s['case']
    kind = case['kind']
    layout = (s['psum'], s['alignment']) if case['experts'] else None
    options = dict(out=s['out']) if case['bound'] else dict(do_zero_padding=True)
    if kind == 'linear':
        return deep_ep.grouped_linear(s['x'], s['w'], layout, **options)
    if kind == 'lora':
        return deep_ep.grouped_lora_linear(s['x'], s['w'], s['a'], s['b'], s['adapter'], layout, scales=s['scales'], **options)
    if kind == 'swiglu':
        return deep_ep.swiglu(s['h'], layout, s['weights'], fused_fp8_quant=case['payload'] == 'fp8', **options)
    if kind == 'linear_train':
        x, w = s['x'].detach().requires_grad_(), s['w'].detach().requires_grad_()
        y = deep_ep.grouped_linear(x, w, layout, **options)
        return (y.detach(), *torch.autograd.grad(y, (x, w), s['grad']))
    h, weights = s['h'].detach().requires_grad_(), s['weights'].detach().requires_grad_()
    a = deep_ep.swiglu(h, layout, weights, **options)
    return (a.detach(), *torch.autograd.grad(a, (h, weights), s['grad']))


def _widen_rows(x):
    if not isinstance(x, tuple):
        return x.float()
    q, scale = x
    return q.float() * scale.repeat_interleave(GROUP, dim=1)[:, :q.size(1)]


def _widen_weights(w):
    if not isinstance(w, tuple):
        return w.float() if w.dim() == 3 else w.float()[None]
    q, scale = w
    return q.float() * scale.repeat_interleave(GROUP, dim=1)[:, :q.size(1)].repeat_interleave(GROUP, dim=2)[:, :, :q.size(2)]


def _by_expert(s, rows):
    """[experts, longest, channels]: every expert's rows, zeros behind its last."""
    return rows[s['table']].masked_fill_(~s['filled'][:, :, None], 0.0)


def _to_rows(s, padded):
    """Back to the layout of the rows, rounded; rows of no expert are zero."""
    return (padded[s['expert'], s['place']] * s['valid'][:, None]).to(torch.bfloat16)


def _gates(s):
    gate, up = s['h'].float().chunk(2, dim=1)
    sigmoid = 1 / (1 + torch.exp(-gate))
    return gate, up, sigmoid


def _plain(s):
    case = s['case']
    kind = case['kind']
    if kind == 'swiglu':
        gate, up, sigmoid = _gates(s)
        a = gate * sigmoid * up * s['weights'][:, None]
        if case['payload'] == 'bf16':
            return a.to(torch.bfloat16)
        q, scale = _quantise_rows(a)
        return q, scale * s['valid'][:, None]
    if kind == 'swiglu_train':
        gate, up, sigmoid = _gates(s)
        silu, weights, grad = gate * sigmoid, s['weights'][:, None], s['grad'].float()
        grad_gate = grad * weights * up * sigmoid * (1 + gate * (1 - sigmoid))
        grad_up = grad * weights * silu
        return (silu * up * weights).to(torch.bfloat16), torch.cat([grad_gate, grad_up], dim=1).to(torch.bfloat16), (grad * silu * up).sum(dim=1)

    x, w = _by_expert(s, _widen_rows(s['x'])), _widen_weights(s['w'])
    y = torch.bmm(x, w.transpose(1, 2))
    if kind == 'lora':
        a, b, adapters, rank = s['a'].float(), s['b'].float(), case['adapters'], case['rank']
        if a.dim() == 3:
            a, b = a[:, None], b[:, None]
        low = torch.bmm(x, a.permute(1, 0, 2, 3).reshape(-1, adapters * rank, case['k']).transpose(1, 2))
        # only what belongs to the row's own adapter goes on
        mine = s['adapter'][s['table']][:, :, None] == torch.arange(adapters, device=DEVICE)
        low = low.view(*low.shape[:2], adapters, rank) * (mine * s['scales'])[:, :, :, None]
        y = y + torch.bmm(low.view(*low.shape[:2], adapters * rank), b.permute(1, 0, 3, 2).reshape(-1, adapters * rank, case['n']))
    if kind != 'linear_train':
        return _to_rows(s, y)
    grad = _by_expert(s, s['grad'].float())
    return _to_rows(s, y), _to_rows(s, torch.bmm(grad, w)), torch.bmm(grad.transpose(1, 2), x).to(torch.bfloat16)


# ---- in 64 bits ---------------------------------------------------------------------------------------

def _exact_rows(x):
    if not isinstance(x, tuple):
        return x.double()
    q, scale = x
    channel = torch.arange(q.size(1), device=DEVICE) // GROUP
    return q.to(torch.float64) * scale.double()[:, channel]


def _exact_weights(w, e):
    if not isinstance(w, tuple):
        return (w[e] if w.dim() == 3 else w).double()
    q, scale = w[0][e], w[1][e].double()
    n, k = (torch.arange(size, device=DEVICE) // GROUP for size in q.shape)
    return q.to(torch.float64) * scale[n][:, k]


def exact(case, seed):
    s = prepare(case, seed)
    counts, start, _, rows = _layout(case, seed)
    kind, k, n = case['kind'], case['k'], case['n']
    if kind.startswith('swiglu'):
        h, weights = s['h'].double(), s['weights'].double()
        gate, up = h[:, :n], h[:, n:]
        sigmoid = torch.sigmoid(gate)
        gated = gate * sigmoid * up
        if kind == 'swiglu_train':
            grad = s['grad'].double()
            slope = sigmoid + gate * sigmoid * torch.sigmoid(-gate)
            by_row = weights.unsqueeze(1) * grad
            grad_h = torch.empty_like(h)
            grad_h[:, :n] = by_row * up * slope
            grad_h[:, n:] = by_row * gate * sigmoid
            return gated * weights.unsqueeze(1), grad_h, torch.linalg.vecdot(grad, gated)
        a = gated * weights.unsqueeze(1)
        if case['payload'] == 'bf16':
            return a
        scale = torch.zeros((rows, -(-n // GROUP)), device=DEVICE, dtype=torch.float64)
        q = torch.zeros_like(a)
        for g in range(scale.size(1)):
            part = a[:, g * GROUP:(g + 1) * GROUP]
            scale[:, g] = torch.clamp(part.abs().max(dim=1).values, min=1e-4) / FP8_MAX
            q[:, g * GROUP:(g + 1) * GROUP] = (part / scale[:, g:g + 1]).to(torch.float8_e4m3fn).double()
        scale[~s['valid']] = 0
        return q, scale

    x = _exact_rows(s['x'])
    y = torch.zeros((rows, n), device=DEVICE, dtype=torch.float64)
    grad_x = torch.zeros((rows, k), device=DEVICE, dtype=torch.float64)
    grad_w = torch.zeros((len(counts), n, k), device=DEVICE, dtype=torch.float64) if kind == 'linear_train' else None
    for e, (c, first) in enumerate(zip(counts, start)):
        mine, w = slice(first, first + c), _exact_weights(s['w'], e)
        y[mine] = x[mine] @ w.t()
        if kind == 'linear_train':
            grad = s['grad'][mine].double()
            grad_x[mine], grad_w[e] = grad @ w, grad.t() @ x[mine]
        for j in range(case['adapters']):
            at = first + torch.nonzero(s['adapter'][mine] == j).squeeze(1)
            a, b = (t[j, e] if case['experts'] else t[j] for t in (s['a'], s['b']))
            y[at] += s['scales'][j].double() * (x[at] @ a.double().t()) @ b.double().t()
    return y if kind != 'linear_train' else (y, grad_x, grad_w)


# ---- what a pass cannot do without ----------------------------------------------------------------------

def work(case):
    counts = _counts(case)
    rows, used, k, n = case['rows'], int((counts > 0).sum()), case['k'], case['n']
    size = 1 if case['payload'] == 'fp8' else 2
    layout = 4 * len(counts)
    if case['kind'] == 'swiglu':
        out = rows * (n + 4 * -(-n // GROUP)) if size == 1 else 2 * rows * n
        return {'bytes': rows * (4 * n + 4) + out + layout, 'flops': 8 * rows * n}
    if case['kind'] == 'swiglu_train':
        # h, gate weights and the result's gradient; the result and the gradients of h and of the gate weights
        return {'bytes': rows * (4 * n + 4 + 2 * n) + rows * (2 * n + 4 * n + 4) + layout, 'flops': 24 * rows * n}
    in_bytes, w_bytes = rows * k * size, used * n * k * size
    if size == 1:
        in_bytes += 4 * rows * -(-k // GROUP)
        w_bytes += 4 * used * -(-n // GROUP) * -(-k // GROUP)
    total, flops = in_bytes + w_bytes + 2 * rows * n + layout, 2 * rows * n * k
    if case['kind'] == 'linear_train':
        # the result's gradient, the gradients of rows and of all experts' weights
        total += 2 * rows * n + 2 * rows * k + 2 * len(counts) * n * k
        flops *= 3
    if case['kind'] == 'lora':
        pairs = int(sum(min(case['adapters'], case['requests'], c) for c in counts))
        total += 2 * pairs * case['rank'] * (k + n) + 4 * rows
        flops += 2 * rows * case['rank'] * (k + n)
    return {'bytes': total, 'flops': flops}
