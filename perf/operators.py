"""The operators over a shard's rows that a model is trained and served with, as
cases that can be timed and checked: the softmax loss of queries over all rows
with its gradients, the quantizer to E4M3 with one scale per block of 128, and
the product of two operands in that form.

``own`` chooses between the plain form (elementary torch operations in FP32,
rounded once at the end) and the package's calls on the same state. Sizes
follow the benchmark's corpora: 128, 768 and 1,024 dimensions, 100,000 rows,
a filter's 1,000,000 of 10M rows, 65,536 list centroids, batches of 1 to 4,096
queries.
"""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
E4M3_MAX = 448.0
BLOCK = 128
TINY = 2.0 ** -100  # the least absmax a block's scale is made from


def listed():
    return [
        # one training pair against a small shard: launches, not bytes
        dict(name='loss-1-1000x128-f32', op='loss', nq=1, rows=1000, dims=128, dtype='f32', scale=0.1, unit=False,
             grad=True),
        # the FP32 corpus of 100,000 rows as the classes of a batch of 1,000
        dict(name='loss-1000-100000x128-f32', op='loss', nq=1000, rows=100000, dims=128, dtype='f32', scale=0.09,
             unit=False, grad=True),
        # the IVF index's centroids as classes: training a router to the lists
        dict(name='loss-4096-65536x768-bf16', op='loss', nq=4096, rows=65536, dims=768, dtype='bf16', scale=20.0,
             unit=True, grad=True),
        # a filter's 1,000,000 halfvec rows as classes of a batch of 1,024
        dict(name='loss-1024-1000000x768-f16', op='loss', nq=1024, rows=1000000, dims=768, dtype='f16', scale=20.0,
             unit=True, grad=True),
        # evaluation of a ragged batch: the loss alone, rows of 402 bytes
        dict(name='loss-77-333333x201-bf16-eval', op='loss', nq=77, rows=333333, dims=201, dtype='bf16', scale=14.0,
             unit=True, grad=False),
        # one query on its way into a scoring call
        dict(name='quant-1x1024-f32', op='quant', m=1, k=1024, dtype='f32', square=False),
        # a halfvec corpus stored as codes
        dict(name='quant-1000000x768-f16', op='quant', m=1000000, k=768, dtype='f16', square=False),
        # a ragged weight matrix in square blocks
        dict(name='quant-65537x1000-bf16-square', op='quant', m=65537, k=1000, dtype='bf16', square=True),
        # one query scored against every row of a shard
        dict(name='product-1x100000x1024-f32', op='product', m=1, n=100000, k=1024, out='f32', square=False),
        # a handful of queries against the list centroids
        dict(name='product-33x65536x768-f32', op='product', m=33, n=65536, k=768, out='f32', square=False),
        # a serving batch's scores over 1,000,000 rows
        dict(name='product-1024x1000000x1024-f16', op='product', m=1024, n=1000000, k=1024, out='f16', square=False),
        # a projection: ragged rows, square blocks on the weight's side
        dict(name='product-8191x5000x4096-bf16', op='product', m=8191, n=5000, k=4096, out='bf16', square=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['loss', 'loss', 'quant', 'product', 'product'])
    if op == 'loss':
        while True:
            nq, rows, dims = _log(rng, 1, 4096), _log(rng, 64, 1000000), _log(rng, 8, 1536)
            if nq * rows * dims <= 3e11 and rows * dims <= 5e8 and nq * rows <= 1e9:
                break
        unit = rng.random() < 0.6
        return dict(op='loss', nq=nq, rows=rows, dims=dims, dtype=rng.choice(['f32', 'f16', 'bf16']), unit=unit,
                    scale=round(rng.uniform(5.0, 25.0) if unit else rng.uniform(0.5, 1.2) / math.sqrt(dims), 4),
                    grad=rng.random() < 0.75)
    if op == 'quant':
        while True:
            m, k = _log(rng, 1, 1000000), _log(rng, 8, 2048)
            if m * k <= 7e8:
                break
        return dict(op='quant', m=m, k=k, dtype=rng.choice(['f32', 'f16', 'bf16']), square=rng.random() < 0.4)
    while True:
        m, n, k = _log(rng, 1, 8192), _log(rng, 1, 1000000), _log(rng, 16, 4096)
        if m * n * k <= 1e12 and m * n <= 1e9 and n * k <= 1e9 and m * n * k >= 1e4:
            break
    return dict(op='product', m=m, n=n, k=k, out=rng.choice(['f32', 'f16', 'bf16']), square=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs

def _corpus(n, d, gen, unit):
    """Rows of a Gaussian mixture, as embeddings are: centres ~N(0, 1), noise 0.1."""
    centres = torch.randn((min(1000, max(1, n // 16)), d), generator=gen, device='cuda')
    x = torch.randn((n, d), generator=gen, device='cuda').mul_(0.1)
    x += centres[torch.randint(0, centres.shape[0], (n,), generator=gen, device='cuda')]
    return x.div_(x.norm(dim=1, keepdim=True).clamp_min(1e-30)) if unit else x


def _codes(m, k, gen, square):
    """An operand in E4M3 with its scales, as it is kept between calls: codes in
    rows of a multiple of 16 bytes, [m, k] of them seen. Made by elementary
    operations, whatever makes it in a user's program."""
    x = _corpus(m, k, gen, False)
    pad = (k + 15) // 16 * 16
    held = torch.zeros((m, pad), dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn)
    codes, scales = _plain_quantize(x, square)
    held[:, :k].view(torch.uint8).copy_(codes.view(torch.uint8))
    return held[:, :k], scales


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    c = dict(case)
    if c['op'] == 'loss':
        dt = DTYPES[c['dtype']]
        w = _corpus(c['rows'], c['dims'], gen, c['unit'])
        t = torch.randint(0, c['rows'], (c['nq'],), generator=gen, device='cuda')
        x = w[t] + torch.randn((c['nq'], c['dims']), generator=gen, device='cuda') * (
            0.5 / math.sqrt(c['dims']) if c['unit'] else 0.5)
        if c['unit']:
            x /= x.norm(dim=1, keepdim=True)
        # a query in twenty has no target: its loss and gradient are zero
        if c['nq'] > 1:
            t[torch.rand((c['nq'],), generator=gen, device='cuda') < 0.05] = -1
        # the mean's weights, times the loss scale that FP16 gradients are kept from vanishing with
        g = (0.5 + torch.rand((c['nq'],), generator=gen, device='cuda')) * (
            (2.0 ** 16 if c['dtype'] == 'f16' else 1.0) / c['nq'])
        return dict(case=c, x=x.to(dt), w=w.to(dt), t=t, g=g)
    if c['op'] == 'quant':
        return dict(case=c, x=_corpus(c['m'], c['k'], gen, True).to(DTYPES[c['dtype']]))
    a, sa = _codes(c['m'], c['k'], gen, False)
    b, sb = _codes(c['n'], c['k'], gen, c['square'])
    return dict(case=c, a=a, sa=sa, b=b, sb=sb)


# ---------------------------------------------------------------- the operators

def _plain_loss(x, w, t, g, scale, grad):
    nq = x.shape[0]
    xf, wf = x.float(), w.float()
    e = (xf @ wf.t()).mul_(scale)
    kept = t >= 0
    at = t.clamp_min(0)
    target = e.gather(1, at[:, None])[:, 0]
    m = e.amax(dim=1)
    e.sub_(m[:, None]).exp_()
    s = e.sum(dim=1)
    lse = m + s.log()
    out = dict(loss=torch.where(kept, lse - target, torch.zeros_like(lse)), lse=lse)
    if grad:
        # the gradient of sum_i g_i loss_i by the logits: g_i (softmax_i - [j = t_i]), zero without a target
        gk = torch.where(kept, g, torch.zeros_like(g))
        e.mul_((gk / s)[:, None])
        e[torch.arange(nq, device=e.device), at] -= gk
        out['dx'] = (e @ wf).mul_(scale).to(x.dtype)
        out['dw'] = (e.t() @ xf).mul_(scale).to(w.dtype)
    return out


def _blocks(x, square):
    """x padded with zeros to whole blocks: [m or mb, 128 or 1, kb, 128]."""
    m, k = x.shape
    kb = (k + BLOCK - 1) // BLOCK
    r = BLOCK if square else 1
    mb = (m + r - 1) // r
    if mb * r != m or kb * BLOCK != k:
        p = torch.zeros((mb * r, kb * BLOCK), dtype=torch.float32, device=x.device)
        p[:m, :k] = x
        x = p
    return x.float().reshape(mb, r, kb, BLOCK)


def _plain_quantize(x, square):
    """scale = absmax / 448 of each block (1 where it is all zeros), code = the
    E4M3 number nearest to x * (448 / absmax), ties to even."""
    m, k = x.shape
    v = _blocks(x, square)
    absmax = v.abs().amax(dim=(1, 3))
    zero = absmax == 0
    made = torch.where(zero, torch.full_like(absmax, E4M3_MAX), absmax.clamp_min(TINY))
    codes = (v * (E4M3_MAX / made)[:, None, :, None]).to(torch.float8_e4m3fn)
    codes = codes.reshape(codes.shape[0] * codes.shape[1], -1)[:m, :k]
    return codes, made / E4M3_MAX


def _decoded(codes, scales, square):
    v = _blocks(codes.float(), square) * scales[:, None, :, None]
    return v.reshape(v.shape[0] * v.shape[1], -1)[:codes.shape[0], :codes.shape[1]]


def run(state):
    c = state['case']
    if own:
        import pgvector_b200 as pb
    if c['op'] == 'loss':
        x, w, t, g = state['x'], state['w'], state['t'], state['g']
        if not own:
            return _plain_loss(x, w, t, g, c['scale'], c['grad'])
        loss, lse = pb.softmax_loss(x, w, t, scale=c['scale'])
        out = dict(loss=loss, lse=lse)
        if c['grad']:
            out['dx'], out['dw'] = pb.softmax_loss_grad(x, w, t, lse, grad=g, scale=c['scale'])
        return out
    if c['op'] == 'quant':
        if own:
            codes, scales = pb.quantize_blocks(state['x'], square=c['square'])
        else:
            codes, scales = _plain_quantize(state['x'], c['square'])
        return dict(codes=codes, scales=scales)
    if own:
        return pb.matmul_blocks(state['a'], state['sa'], state['b'], state['sb'], dtype=DTYPES[c['out']])
    a = _decoded(state['a'], state['sa'], False)
    b = _decoded(state['b'], state['sb'], c['square'])
    return (a @ b.t()).to(DTYPES[c['out']])


def work(case):
    size = {'f32': 4, 'f16': 2, 'bf16': 2}
    if case['op'] == 'loss':
        e = size[case['dtype']]
        held = (case['nq'] + case['rows']) * case['dims'] * e
        small = case['nq'] * (8 + 4 + 4)
        product = 2.0 * case['nq'] * case['rows'] * case['dims']
        # the logits, and with the gradient one product more for each side
        return {'bytes': held + small + (held + 4 * case['nq'] if case['grad'] else 0),
                'flops': product * (3 if case['grad'] else 1)}
    if case['op'] == 'quant':
        kb = (case['k'] + BLOCK - 1) // BLOCK
        mb = (case['m'] + BLOCK - 1) // BLOCK if case['square'] else case['m']
        return {'bytes': case['m'] * case['k'] * (size[case['dtype']] + 1) + 4 * mb * kb,
                'flops': 2.0 * case['m'] * case['k']}
    kb = (case['k'] + BLOCK - 1) // BLOCK
    nb = (case['n'] + BLOCK - 1) // BLOCK if case['square'] else case['n']
    return {'bytes': (case['m'] + case['n']) * case['k'] + 4 * kb * (case['m'] + nb)
            + case['m'] * case['n'] * size[case['out']],
            'flops': 2.0 * case['m'] * case['n'] * case['k']}


# ---------------------------------------------------------------- from the definitions, in 64 bits

def _exact_loss(x, w, t, g, scale, grad, piece=65536):
    x, w, g = x.double(), w.double(), g.double()
    nq, n = x.shape[0], w.shape[0]
    logit = torch.cat([x @ w[i:i + piece].t() * scale for i in range(0, n, piece)], dim=1)
    lse = torch.logsumexp(logit, dim=1)
    has = (t >= 0).double()
    loss = torch.zeros_like(lse)
    at = torch.nonzero(t >= 0)[:, 0]
    loss[at] = lse[at] - logit[at, t[at]]
    out = dict(loss=loss, lse=lse)
    if grad:
        dx, dw = torch.zeros_like(x), []
        for i in range(0, n, piece):
            p = torch.exp(logit[:, i:i + piece] - lse[:, None])
            inside = torch.nonzero((t >= i) & (t < i + p.shape[1]))[:, 0]
            p[inside, t[inside] - i] -= 1.0
            p *= (has * g * scale)[:, None]
            dx += p @ w[i:i + piece]
            dw.append(p.t() @ x)
        out['dx'], out['dw'] = dx, torch.cat(dw)
    return out


def _exact_quantize(x, square):
    m, k = x.shape
    x = x.double()
    v = torch.nn.functional.pad(x, (0, -k % BLOCK, 0, (-m % BLOCK) if square else 0))
    r = BLOCK if square else 1
    absmax = v.abs().reshape(-1, r, v.shape[1] // BLOCK, BLOCK).permute(0, 2, 1, 3).reshape(
        v.shape[0] // r, v.shape[1] // BLOCK, -1).max(dim=2).values
    scales = torch.where(absmax > 0, absmax.clamp_min(TINY) / E4M3_MAX, torch.ones_like(absmax))
    # the step of E4M3 at |u|: 2^(exponent - 3), at least 2^-9; the nearest multiple, ties to even
    u = x / scales.repeat_interleave(r, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3.0)
    return dict(codes=(torch.round(u / step) * step).clamp(-E4M3_MAX, E4M3_MAX), scales=scales)


def _exact_product(a, sa, b, sb, square, piece=131072):
    a = a.float().double() * sa.double().repeat_interleave(BLOCK, 1)[:, :a.shape[1]]
    out = []
    for i in range(0, b.shape[0], piece):
        s = sb[i // BLOCK:(i + piece) // BLOCK].repeat_interleave(BLOCK, 0) if square else sb[i:i + piece]
        q = b[i:i + piece].float().double()
        out.append(a @ (q * s[:q.shape[0]].double().repeat_interleave(BLOCK, 1)[:, :q.shape[1]]).t())
    return torch.cat(out, dim=1)


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'loss':
        return _exact_loss(s['x'], s['w'], s['t'], s['g'], case['scale'], case['grad'])
    if case['op'] == 'quant':
        return _exact_quantize(s['x'], case['square'])
    return _exact_product(s['a'], s['sa'], s['b'], s['sb'], case['square'])
