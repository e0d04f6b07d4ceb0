"""The serving operators of the decoder's output side: what is measured, in plain form and through the package.

Three operators that a decoding service runs behind the recurrence, one after the other:

  product   y = sa[m] * sw[n] * sum_k qa[m][k] * qw[n][k] (+ bias[n]): operands in 8-bit integers, a scale for each row of
            activations (token) and each row of weights (output channel)
  linear    the same from activations as the layer in front leaves them: every row is quantised (symmetric, its largest magnitude
            becomes 127, ties to even) and multiplied, one call
  sample    a token a row from its logits and ONE given uniform number: temperature, then the top-k largest, then the smallest
            prefix of those that reaches top-p of their mass, then min-p of the largest probability; in what is left the first token,
            in the order of the vocabulary, whose running sum passes u times the whole.  Equal logits rank by index.

`own` False: plain torch operations.  `own` True: the package's calls.  Sizes are those of this repository's configurations (decoder
states of 800 and 2048, a vocabulary of 1806, 256 utterances, 34 x 256 rows of a sequence) and round ones of larger models."""
import math

import numpy as np
import torch

own = False

_DT = {'f32': torch.float32, 'bf16': torch.bfloat16}
_TOP = float(np.finfo(np.float32).max)


def listed():
    return [
        # one utterance's decoder state against the vocabulary: the call whose latency a spoken word waits for
        dict(name='product-state-vocab', op='product', M=1, N=1806, K=800, out='f32', bias=True),
        # a decode batch of 256 utterances against the vocabulary
        dict(name='product-batch-vocab', op='product', M=256, N=1806, K=800, out='f32', bias=True),
        # sixteen streams through a large layer: bound by the weights' bytes
        dict(name='product-16-rows-wide', op='product', M=16, N=16384, K=8192, out='bf16', bias=False),
        # a whole sequence's input projection, 34 steps x 256 utterances; 801 columns: no whole number of tiles
        dict(name='product-sequence-odd', op='product', M=8704, N=3200, K=801, out='bf16', bias=False),
        # the same of the large configuration
        dict(name='product-sequence-large', op='product', M=8704, N=8192, K=2048, out='bf16', bias=True),
        # one token through a square layer, activations quantised on the way
        dict(name='linear-one-token', op='linear', M=1, N=4096, K=4096, x='bf16', out='bf16', bias=False),
        # two dozen hypotheses of a search against the vocabulary
        dict(name='linear-beam-vocab', op='linear', M=24, N=1806, K=2048, x='bf16', out='f32', bias=True),
        # a long batch of fp32 activations, ragged in every size
        dict(name='linear-batch-ragged', op='linear', M=4099, N=4100, K=4104, x='f32', out='bf16', bias=True),
        # one utterance's next word
        dict(name='sample-one-small', op='sample', B=1, V=1806, x='f32', rows='all', masked=0),
        # a decode batch, every row with settings of its own (greedy rows among them)
        dict(name='sample-batch-small', op='sample', B=256, V=1806, x='f32', rows='mixed', masked=3),
        # a few streams over a large vocabulary, half of it masked by a grammar
        dict(name='sample-few-large', op='sample', B=4, V=131072, x='bf16', rows='nucleus', masked=65536),
        # a full batch over a large, odd vocabulary, every row with settings of its own
        dict(name='sample-batch-large', op='sample', B=256, V=128003, x='f32', rows='mixed', masked=17),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['product', 'linear', 'sample'])
    if op == 'sample':
        while True:
            B, V = _log(rng, 1, 512), _log(rng, 2, 262144)
            if B * V <= 256 * 128003:
                break
        return dict(op=op, B=B, V=V, x=rng.choice(['f32', 'bf16']), rows=rng.choice(['all', 'mixed', 'nucleus', 'plain', 'k']),
                    masked=rng.choice([0, rng.randrange(V), min(V - 1, 5)]))
    while True:
        M, N, K = _log(rng, 1, 8704), _log(rng, 50, 16384), _log(rng, 24, 16384)
        if M * N * K <= 8704 * 8192 * 2048 and max(M, N) * K <= 16384 * 8192:
            break
    return dict(op=op, M=M, N=N, K=K, out=rng.choice(['f32', 'bf16']), bias=rng.random() < 0.5,
                **({} if op == 'product' else dict(x=rng.choice(['f32', 'bf16']))))


def _settings(rows, B, g):
    """Per-row sampling settings (temperature, top_k, top_p, min_p) as fp32 / int32 tensors of B."""
    r = torch.rand(4, B, generator=g)
    t = 0.6 + 0.8 * r[0]
    k = torch.zeros(B, dtype=torch.int32)
    p = torch.ones(B)
    m = torch.zeros(B)
    if rows in ('all', 'k'):
        k[:] = (1 + 200 * r[1]).to(torch.int32)
    if rows in ('all', 'nucleus'):
        p = 0.8 + 0.19 * r[2]
    if rows == 'all':
        m = 0.02 * r[3]
    if rows == 'mixed':
        i = torch.arange(B)
        t = torch.where(i % 7 == 3, torch.zeros(()), t)
        k = torch.where(i % 2 == 0, (1 + 100 * r[1]).to(torch.int32), k)
        p = torch.where(i % 3 != 0, 0.7 + 0.29 * r[2], p)
        m = torch.where(i % 5 == 0, 0.05 * r[3], m)
    return t, k, p, m


def _quantised(x):
    """Rows of x (float64) in 8 bits: whole numbers (int8) and the fp32 scale of each row."""
    top = x.abs().amax(1, keepdim=True)
    q = torch.where(top > 0, torch.round(x * 127 / torch.where(top > 0, top, torch.ones_like(top))), torch.zeros_like(x))
    return q.to(torch.int8), (top[:, 0] / 127).float()


def _int8_rows(rows, cols, g, dev):
    """A quantised matrix as it lies in memory: rows zero-padded to a multiple of 64 columns, and its scales."""
    ld = (cols + 63) // 64 * 64
    q = torch.zeros(rows, ld, dtype=torch.int8, device=dev)
    scale = torch.empty(rows, device=dev)
    step = max(1, (1 << 25) // cols)
    for a in range(0, rows, step):
        x = torch.randn(min(step, rows - a), cols, generator=g, device=dev) * 0.05
        q[a:a + step, :cols], scale[a:a + step] = _quantised(x.double())
    return q, scale


def prepare(case, seed):
    dev = torch.device('cuda', torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    c = dict(case)
    if c['op'] == 'sample':
        cpu = torch.Generator()
        cpu.manual_seed(seed)
        B, V = c['B'], c['V']
        # a language model's rows: a wide bulk and a few tokens that stand out
        l = 2.0 * torch.randn(B, V, generator=g, device=dev)
        hot = torch.randint(0, V, (B, 12), generator=g, device=dev)
        l.scatter_add_(1, hot, 6.0 + 3.0 * torch.randn(B, 12, generator=g, device=dev))
        if c['masked']:
            start = int(torch.randint(0, V, (1,), generator=cpu))
            l[:, (torch.arange(c['masked'], device=dev) + start) % V] = float('-inf')
        t, k, p, m = _settings(c['rows'], B, cpu)
        return dict(case=c, logits=l.to(_DT[c['x']]), u=torch.rand(B, generator=cpu).to(dev), temperature=t.to(dev), top_k=k.to(dev),
                    top_p=p.to(dev), min_p=m.to(dev))
    M, N, K = c['M'], c['N'], c['K']
    s = dict(case=c, bias=torch.randn(N, generator=g, device=dev) if c['bias'] else None)
    s['qw'], s['sw'] = _int8_rows(N, K, g, dev)
    if c['op'] == 'product':
        s['qa'], s['sa'] = _int8_rows(M, K, g, dev)
    else:
        s['x'] = torch.randn(M, K, generator=g, device=dev).to(_DT[c['x']])
    return s


def _product(qa, sa, qw, sw, bias, out):
    y = (qa.float() @ qw.float().t()) * sa[:, None] * sw[None, :]
    return (y if bias is None else y + bias).to(out)


def _sample(s):
    # (in 64 bits: a running sum over a large vocabulary lies next to u times the whole more often than 32 bits can tell)
    l = s['logits'].double()
    l = torch.where(torch.isnan(l), torch.full_like(l, -math.inf), l).clamp(max=_TOP)
    B, V = l.shape
    v, order = torch.sort(l, dim=1, descending=True, stable=True)
    t = s['temperature'].double()[:, None]
    greedy = t <= 0
    x = (v - v[:, :1]) / torch.where(greedy, torch.ones_like(t), t)
    w = torch.exp(x)
    k = s['top_k'].long()[:, None]
    keep = (v > -math.inf) & ((torch.arange(V, device=l.device)[None] < k) | (k <= 0))
    w = torch.where(keep, w, torch.zeros_like(w))
    run = torch.cumsum(w, 1)
    p = s['top_p'].double()[:, None]
    keep = keep & ((run - w < p * run[:, -1:]) | (p >= 1)) & (w >= s['min_p'].double()[:, None])
    w = torch.where(keep, w, torch.zeros_like(w))
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    run = torch.cumsum(by_index, 1)
    total = run[:, -1:]
    token = (run > s['u'].double()[:, None] * total).to(torch.int8).argmax(1, keepdim=True)
    token = torch.where(greedy, order[:, :1], token)
    logprob = (l.gather(1, token) - v[:, :1]) / torch.where(greedy, torch.ones_like(t), t) - torch.log(total)
    logprob = torch.where(greedy, torch.zeros_like(logprob), logprob)
    return token[:, 0].int(), logprob[:, 0].float()


def run(state):
    c = state['case']
    if own:
        from ecog2txt_amd import serving
        if c['op'] == 'sample':
            return serving.sample_rows(state['logits'], state['u'], temperature=state['temperature'], top_k=state['top_k'],
                                       top_p=state['top_p'], min_p=state['min_p'])
        w = serving.Int8Rows(state['qw'], state['sw'], c['K'])
        if c['op'] == 'product':
            return serving.matmul_i8(serving.Int8Rows(state['qa'], state['sa'], c['K']), w, bias=state['bias'], out_dtype=_DT[c['out']])
        return serving.linear_i8(state['x'], w, bias=state['bias'], out_dtype=_DT[c['out']])
    if c['op'] == 'sample':
        return _sample(state)
    if c['op'] == 'product':
        return _product(state['qa'], state['sa'], state['qw'], state['sw'], state['bias'], _DT[c['out']])
    q, scale = _quantised(state['x'].double())       # (64 bits: whole numbers next to a border of the rounding)
    return _product(q, scale, state['qw'][:, :c['K']], state['sw'], state['bias'], _DT[c['out']])


def work(case):
    c = case
    if c['op'] == 'sample':
        n = c['B'] * c['V']
        return dict(bytes=n * (4 if c['x'] == 'f32' else 2) + c['B'] * 28, flops=n * 4)
    M, N, K = c['M'], c['N'], c['K']
    a = M * K + 4 * M if c['op'] == 'product' else M * K * (4 if c['x'] == 'f32' else 2)
    return dict(bytes=a + N * K + 4 * N + (4 * N if c['bias'] else 0) + M * N * (4 if c['out'] == 'f32' else 2), flops=2 * M * N * K)


def _exact_row(l, u, t, k, p, m):
    """One row from the definition, float64 numpy: (token, log-probability)."""
    l = np.minimum(np.where(np.isnan(l), -np.inf, l), _TOP)
    if t <= 0:
        return int(np.argmax(l)), 0.0
    rank = np.argsort(-l, kind='stable')
    rank = rank[:np.count_nonzero(l > -np.inf)]
    w = np.exp((l[rank] - l[rank[0]]) / t)
    n = len(rank) if k <= 0 else min(int(k), len(rank))
    if p < 1:
        mass = np.cumsum(w[:n])
        n = min(n, max(1, int(np.searchsorted(mass, p * mass[-1])) + 1))
    n = min(n, max(1, int(np.searchsorted(-w, -m, side='right')))) if m > 0 else n
    left = np.sort(rank[:n])
    w = np.exp((l[left] - l[rank[0]]) / t)
    mass = np.cumsum(w)
    i = min(int(np.searchsorted(mass, u * mass[-1], side='right')), n - 1)
    return int(left[i]), float((l[left[i]] - l[rank[0]]) / t - np.log(mass[-1]))


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'sample':
        host = [s[n].double().cpu().numpy() for n in ('logits', 'u', 'temperature', 'top_k', 'top_p', 'min_p')]
        got = [_exact_row(*row) for row in zip(*host)]
        return np.array([r[0] for r in got], np.int32), np.array([r[1] for r in got], np.float64)
    K = case['K']
    w, sw = s['qw'][:, :K].double(), s['sw'].double()
    if case['op'] == 'product':
        a, sa = s['qa'][:, :K].double(), s['sa'].double()
    else:
        x = s['x'].double()
        top = x.abs().max(1, keepdim=True).values
        a, sa = torch.round(127 * x / top), top[:, 0] / 127
    y = torch.mul(torch.mm(a, w.t()), torch.outer(sa, sw))
    return y if s['bias'] is None else y + s['bias'].double()
