"""What the 8-bit operators of the framework are measured on: the block quantiser, the block-scaled products (serving,
batches, training) and the AdamW step over many tensors with its states in 32 or in 8 bits.

`own = False`: every operator in elementary torch operations; `own = True`: the framework's entry points
(`conv1d_text_vae_amd.fp8`, `conv1d_text_vae_amd.optim`) on the same inputs.
"""
import math

import torch
import torch.nn.functional as F

own = False

DEV = 'cuda' if torch.cuda.is_available() else 'cpu'
BLOCK = 128                     # elements that share a scale
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the word vectors of one served batch (64 texts of 16 words, 302 values) going into the generator
        dict(name='quantize_words', op='quantize', rows=1024, cols=302, gap=0, type='f32', both=False),
        # activations of a training step, needed along the row (forward) and along the column (weight gradient)
        dict(name='quantize_train', op='quantize', rows=16384, cols=2048, gap=0, type='bf16', both=True),
        # one character of one text: the state times a recurrent kernel of 1024 units (latency)
        dict(name='dense_one_text', op='dense', rows=1, k=1024, n=1024, gap=0, type='f32', bias=True, relu=False),
        # 13 texts at once against a large layer: the weights' bytes decide
        dict(name='dense_13_texts', op='dense', rows=13, k=4096, n=8192, gap=0, type='bf16', bias=True, relu=False),
        # the two latent heads of a batch of 256: [256, 1920] x [1920, 512]
        dict(name='dense_heads', op='dense', rows=256, k=1920, n=512, gap=0, type='f32', bias=True, relu=False),
        # an odd batch of 302-wide word vectors (rows 305 values apart) onto an odd number of outputs
        dict(name='dense_ragged', op='dense', rows=1999, k=302, n=1021, gap=3, type='bf16', bias=True, relu=True),
        # both operands quantised before: the product alone at the size where the matrix units decide
        dict(name='product_large', op='product', rows=8192, k=8192, n=8192, type='bf16'),
        # input projection of the generator in a training step, forward and backward: 128 texts of 16 words, 1024 units
        dict(name='linear_words', op='linear', rows=2048, k=302, n=1024, type='f32', bias=True),
        # a wide layer in training, forward and backward
        dict(name='linear_wide', op='linear', rows=16384, k=2048, n=4096, type='bf16', bias=True),
        # the generator with 128 units: a dozen small tensors, global-norm clip (latency)
        dict(name='adamw_generator', op='adamw', tensors=12, n=200000, states='f32', grads='f32', clip=10.0, seed=3),
        # 160 million weights in 40 tensors, no clip
        dict(name='adamw_wide', op='adamw', tensors=40, n=160000000, states='f32', grads='f32', clip=0.0, seed=4),
        # the same number of weights with states in 8 bits, bf16 gradients and the clip
        dict(name='adamw8_wide', op='adamw', tensors=40, n=160000000, states='8bit', grads='bf16', clip=10.0, seed=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['quantize', 'dense', 'dense', 'product', 'linear', 'adamw', 'adamw'])
    kind = rng.choice(['f32', 'bf16'])
    if op == 'quantize':
        rows = _log(rng, 1, 16384)
        return dict(op=op, rows=rows, cols=_log(rng, 1, min(8192, 33554432 // rows)), gap=rng.choice([0, 0, 1, 8]), type=kind,
                    both=rng.random() < 0.5)
    if op == 'dense':
        return dict(op=op, rows=rng.choice([_log(rng, 1, 16), _log(rng, 17, 4096)]), k=_log(rng, 16, 8192), n=_log(rng, 8, 8192),
                    gap=rng.choice([0, 0, 3, 8]), type=kind, bias=rng.random() < 0.7, relu=rng.random() < 0.3)
    if op == 'product':
        return dict(op=op, rows=_log(rng, 64, 8192), k=_log(rng, 64, 8192), n=_log(rng, 64, 8192), type=kind)
    if op == 'linear':
        return dict(op=op, rows=_log(rng, 1, 16384), k=_log(rng, 8, 2048), n=_log(rng, 8, 4096), type=kind, bias=rng.random() < 0.7)
    return dict(op=op, tensors=rng.randint(1, 48), n=_log(rng, 1000, 100000000), states=rng.choice(['f32', '8bit']),
                grads=rng.choice(['f32', 'bf16']), clip=rng.choice([0.0, 1.0, 10.0]), seed=rng.randint(0, 1 << 30))


def _sizes(case):
    """Element counts of an optimizer case: the first two thirds are matrices (decayed), the others vectors (not decayed);
    odd counts among them, and they add up to about `n`."""
    import random
    rng = random.Random(case['seed'])
    t = case['tensors']
    mats = max(1, (2 * t + 2) // 3)
    share = [math.exp(rng.uniform(0.0, 3.0)) for _ in range(mats)]
    total = sum(share)
    sizes = []
    for s in share:
        rows = max(1, int(math.sqrt(case['n'] * s / total)))
        cols = max(1, int(case['n'] * s / total / rows))
        sizes.append((rows, cols))
    sizes += [(rng.randint(1, 4096),) for _ in range(t - mats)]
    return sizes, mats


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _activations(gen, rows, cols, kind, gap=0):
    """Rows of different magnitude, a few large values, one row in ten empty (behind the end of a text); `gap` values lie
    between the rows."""
    x = _normal(gen, rows, cols)
    x *= torch.exp(_normal(gen, rows, 1))
    x = torch.where(torch.rand(rows, cols, generator=gen, device=DEV) < 1e-3, x * 30, x)
    if rows > 1:
        x *= (torch.rand(rows, 1, generator=gen, device=DEV) >= 0.1)
    x = x.to(TYPES[kind])
    if not gap:
        return x
    wide = torch.zeros(rows, cols + gap, dtype=x.dtype, device=DEV)
    wide[:, :cols] = x
    return wide[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1000003 * (seed + 1))
    op = case['op']
    s = dict(case=case)
    if op == 'quantize':
        s['x'] = _activations(gen, case['rows'], case['cols'], case['type'], case['gap'])
    elif op == 'dense':
        s['x'] = _activations(gen, case['rows'], case['k'], case['type'], case['gap'])
        w = _normal(gen, case['n'], case['k']) / math.sqrt(case['k'])
        s['w'] = _blocks(w)                                     # a served layer keeps its weights in 8 bits
        s['bias'] = _normal(gen, case['n']) if case['bias'] else None
    elif op == 'product':
        s['a'] = _blocks(_activations(gen, case['rows'], case['k'], 'f32'))
        s['b'] = _blocks(_normal(gen, case['n'], case['k']) / math.sqrt(case['k']))
    elif op == 'linear':
        s['x'] = _activations(gen, case['rows'], case['k'], case['type']).requires_grad_(True)
        s['kernel'] = (_normal(gen, case['k'], case['n']) / math.sqrt(case['k'])).requires_grad_(True)
        s['bias'] = (0.1 * _normal(gen, case['n'])).requires_grad_(True) if case['bias'] else None
        s['dy'] = (1e-3 * _activations(gen, case['rows'], case['n'], 'f32')).to(TYPES[case['type']])
    else:
        _prepare_adamw(s, case, gen)
    return s


def _prepare_adamw(s, case, gen):
    """An optimizer in the middle of a run: 99 steps done.  Every tensor's state begins at a whole block of one flat buffer."""
    sizes, mats = _sizes(case)
    s['lr'], s['betas'], s['eps'] = 1e-3, (0.9, 0.999), 1e-8
    s['wd'] = [0.01] * mats + [0.0] * (len(sizes) - mats)
    s['params'], s['grads'], at = [], [], []
    end = 0
    for shape in sizes:
        p = _normal(gen, *shape) * 0.02
        g = _normal(gen, *shape) * torch.exp(2 * torch.randn(1, generator=gen, device=DEV)) * 1e-3
        s['params'].append(p)
        s['grads'].append(g.to(TYPES[case['grads']]))
        at.append((end, p.numel()))
        end += -(-p.numel() // BLOCK) * BLOCK
    s['decayed'] = at[mats][0] if mats < len(at) else end
    s['work'] = torch.zeros(end, device=DEV)
    s['views'] = [s['work'][a:a + n].view(shape) for (a, n), shape in zip(at, sizes)]
    # momenta: the gradient's magnitude, each value with its own spread
    torch._foreach_copy_(s['views'], s['grads'])
    spread = torch.exp(0.5 * _normal(gen, end))
    v = s['work'].square() * spread
    m = s['work'] * (0.3 * _normal(gen, end))
    s['step'] = torch.tensor([99], dtype=torch.int64, device=DEV)
    s['rng_seed'] = int(case['seed']) * 7 + 1
    if case['states'] == 'f32':
        s['m'], s['v'], s['m_scale'], s['v_scale'] = m, v, None, None
    else:
        half = torch.full((end,), 1 << 15, dtype=torch.int32, device=DEV)
        s['m'], s['m_scale'] = _pack_m(m, half)
        s['v'], s['v_scale'] = _pack_v(v, half)
    if own:      # the handle that a program keeps beside its parameters
        from conv1d_text_vae_amd import optim
        s['opt'] = optim.AdamW(s['params'], lr=s['lr'], betas=s['betas'], eps=s['eps'], weight_decay=s['wd'],
                               clipnorm=case['clip'], states=case['states'], seed=s['rng_seed'])
        s['opt'].load_state_dict({k: s[k] for k in ('step', 'm', 'v', 'm_scale', 'v_scale')})


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _blocks(x):
    """[R, C] -> (e4m3 values [R, Cp], scale bytes [Cp / 128, R rounded up to 16]): value = q * 2^(s - 127), 2^(s - 127) the
    smallest power of two, 2^-111 at least, that keeps the block's largest finite magnitude at 448 or less; 127 behind the
    last row."""
    rows, cols = x.shape
    x = F.pad(x.float(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    finite = torch.isfinite(x)
    amax = torch.where(finite, x.abs(), 0.0).amax(-1)
    frac, expo = torch.frexp(amax)                              # amax = frac * 2^expo, frac in [1/2, 1); 448 = 7/8 * 2^9
    s = torch.where(amax > 0, expo - 9 + (frac > 0.875) + 127, 127).clamp(16, 254)
    q = x * _power(254 - s).unsqueeze(-1)
    q = torch.where(finite, q, float('nan')).to(torch.float8_e4m3fn)
    return q.view(rows, -1), F.pad(s.t(), (0, -rows % 16), value=127).to(torch.uint8)


def _power(s):
    """2^(s - 127) as float32, 1 <= s <= 254."""
    return (s.to(torch.int32) << 23).view(torch.float32)


def _values(q, s):
    return (q.float().view(q.shape[0], -1, BLOCK) * _power(s[:, :q.shape[0]]).t().unsqueeze(-1)).view(q.shape)


def _product(a, b, bias=None, relu=False, kind=torch.float32):
    y = _values(*a) @ _values(*b).t()
    if bias is not None:
        y = y + bias
    return (torch.relu(y) if relu else y).to(kind)


def _linear(x, kernel, bias, dy):
    kind = x.dtype
    x, kernel, dy = x.detach(), kernel.detach(), dy.detach()
    out = dict(y=_product(_blocks(x), _blocks(kernel.t()), None if bias is None else bias.detach(), kind=kind))
    out['dx'] = _product(_blocks(dy), _blocks(kernel), kind=kind)
    out['dkernel'] = _product(_blocks(x.t()), _blocks(dy.t()))
    if bias is not None:
        out['dbias'] = dy.float().sum(0)
    return out


def _philox_halves(n, seed, step):
    """16 random bits for each of n elements: Philox4x32-10 with counter (block, block >> 32, step, step >> 32) and key `seed`;
    element e takes half-word e & 7 of block e >> 3."""
    mask = 0xFFFFFFFF
    blk = torch.arange(n // 8, dtype=torch.int64, device=DEV)
    c = [blk & mask, blk >> 32, torch.full_like(blk, step & mask), torch.full_like(blk, step >> 32)]
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((p1 >> 32) & mask) ^ c[1] ^ k0, p1 & mask, ((p0 >> 32) & mask) ^ c[3] ^ k1, p0 & mask]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], dim=1).view(-1).to(torch.int32)


def _block_exponent(x):
    """Biased exponent (as in float32) of the largest finite magnitude of each block of x [n]."""
    x = torch.where(torch.isfinite(x), x, 0.0).view(-1, BLOCK).amax(1)
    return x.view(torch.int32) >> 23


def _pack_m(m, r):
    """m -> e4m3 values and scale bytes; the largest magnitude of a block lies in [128, 256) of its scale, the bits behind
    the third of the mantissa are rounded up with the probability that they stand for (r: 16 random bits)."""
    s = (_block_exponent(m.abs()) - 7).clamp(min=1)
    x = (m.abs().view(-1, BLOCK) * _power(254 - s).unsqueeze(1)).view(-1)
    small = x < 2.0 ** -6                                       # below the normal numbers the steps are even
    bits = torch.where(small, x + 2.0 ** -6, x).view(torch.int32) + ((r << 4) | 8)
    c = (bits >> 20) - (121 << 3) + torch.where(small, 0, 8)
    c = torch.where(torch.isfinite(m), c, 0x7F) | torch.where(torch.signbit(m), 0x80, 0)
    return c.to(torch.uint8).view(torch.float8_e4m3fn), s.to(torch.uint8)


def _pack_v(v, r):
    """v >= 0 -> a byte of five exponent and three mantissa bits and scale bytes: 0 is zero, 255 is NaN, c stands for the
    float32 with bits (c + 8 s - 240) << 20; what is not zero stays at 1 or more."""
    s = _block_exponent(v).clamp(min=32)
    r = (r * 40503) & 0xFFFF
    base = (8 * s - 240).unsqueeze(1)
    c = ((v.view(torch.int32) + ((r << 4) | 8)) >> 20).view(-1, BLOCK) - base
    c = torch.where(v > 0, c.view(-1).clamp(min=1), 0)
    return torch.where(torch.isfinite(v), c, 255).to(torch.uint8), s.to(torch.uint8)


def _unpack_v(c, s):
    b = c.to(torch.int32).view(-1, BLOCK) + (8 * s.to(torch.int32) - 240).unsqueeze(1)
    v = (b << 20).view(torch.float32).view(-1)
    return torch.where(c == 0, 0.0, torch.where(c == 255, float('nan'), v))


def _adamw(s):
    case, g = s['case'], s['work']
    b1, b2 = s['betas']
    s['step'] += 1
    s['done'] = t = s.get('done', 99) + 1                       # the step number on the host's side
    torch._foreach_copy_(s['views'], s['grads'])
    if case['clip'] > 0:
        norm = g.double().square().sum().sqrt().float()         # a long sum: in 64 bits
        g.mul_(torch.where(norm >= case['clip'], case['clip'] / norm, 1.0))
    e8 = case['states'] == '8bit'
    m = (_values(s['m'].view(-1, BLOCK), s['m_scale'].view(1, -1)).view(-1) if e8 else s['m'])
    v = _unpack_v(s['v'], s['v_scale']) if e8 else s['v']
    m.mul_(b1).add_(g * (1.0 - b1))
    v.mul_(b2).add_(g.square() * (1.0 - b2))
    d = (v / (1.0 - b2 ** t)).sqrt_().add_(s['eps'])
    d = torch.div(m, d, out=d).mul_(s['lr'] / (1.0 - b1 ** t))
    torch._foreach_copy_(s['views'], s['params'])
    g[:s['decayed']].mul_(1.0 - s['lr'] * s['wd'][0])
    g.sub_(d)
    torch._foreach_copy_(s['params'], s['views'])
    if e8:
        r = _philox_halves(g.numel(), s['rng_seed'], t)
        q, qs = _pack_m(m, r)
        s['m'].copy_(q), s['m_scale'].copy_(qs)
        q, qs = _pack_v(v, r)
        s['v'].copy_(q), s['v_scale'].copy_(qs)
    return dict(params=s['params'], m=s['m'], v=s['v'], step=s['step'],
                **(dict(m_scale=s['m_scale'], v_scale=s['v_scale']) if e8 else {}), **(dict(norm=norm) if case['clip'] > 0 else {}))


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_plain(s):
    case = s['case']
    op = case['op']
    if op == 'quantize':
        return [*_blocks(s['x']), *(_blocks(s['x'].t()) if case['both'] else ())]
    if op == 'dense':
        return _product(_blocks(s['x']), s['w'], s['bias'], case['relu'], s['x'].dtype)
    if op == 'product':
        return _product(s['a'], s['b'], kind=TYPES[case['type']])
    if op == 'linear':
        return _linear(s['x'], s['kernel'], s['bias'], s['dy'])
    return _adamw(s)


def _run_own(s):
    from conv1d_text_vae_amd import fp8
    case = s['case']
    op = case['op']
    if op == 'quantize':
        got = fp8.quantize_both(s['x']) if case['both'] else (fp8.quantize_rows(s['x']),)
        return [t for q in got for t in (q.data, q.scale)]
    if op == 'dense':
        return fp8.dense(s['x'], fp8.Fp8Rows(*s['w'], case['k']), s['bias'], relu=case['relu'])
    if op == 'product':
        return fp8.product(fp8.Fp8Rows(*s['a'], case['k']), fp8.Fp8Rows(*s['b'], case['k']), out_dtype=TYPES[case['type']])
    if op == 'linear':
        leaves = [s['x'], s['kernel']] + ([s['bias']] if s['bias'] is not None else [])
        y = fp8.linear(s['x'], s['kernel'], s['bias'])
        grads = torch.autograd.grad(y, leaves, s['dy'])
        return dict(zip(('y', 'dx', 'dkernel', 'dbias'), (y.detach(), *grads)))
    opt = s['opt']
    opt.step(s['grads'])
    return dict(params=s['params'], m=opt.m, v=opt.v, step=opt.t,
                **(dict(m_scale=opt.m_scale, v_scale=opt.v_scale) if case['states'] == '8bit' else {}),
                **(dict(norm=opt.norm) if case['clip'] > 0 else {}))


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    op = case['op']
    up = lambda n: -(-n // BLOCK) * BLOCK
    size = {'f32': 4, 'bf16': 2}
    q = 1 + 1 / BLOCK                                           # bytes of a value and its share of the scale
    if op == 'quantize':
        r, c = case['rows'], case['cols']
        return dict(bytes=r * c * size[case['type']] + r * up(c) * q + (c * up(r) * q if case['both'] else 0), flops=2 * r * c)
    if op == 'adamw':
        n = sum(math.prod(shape) for shape in _sizes(case)[0])
        state = 16 if case['states'] == 'f32' else 4 * q
        return dict(bytes=n * (8 + state + size[case['grads']]), flops=16 * n)
    m, k, n, e = case['rows'], case['k'], case['n'], size[case['type']]
    if op == 'dense':
        return dict(bytes=m * k * e + n * up(k) * q + m * n * e + (4 * n if case['bias'] else 0), flops=2 * m * n * k)
    if op == 'product':
        return dict(bytes=(m + n) * up(k) * q + m * n * e, flops=2 * m * n * k)
    return dict(bytes=2 * m * k * e + 2 * k * n * 4 + 2 * m * n * e + (8 * n if case['bias'] else 0), flops=6 * m * n * k)


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _nearest_blocks(x):
    """The quantised values in units of their scales, and the scales' exponents, from the definition."""
    rows, cols = x.shape
    x = F.pad(x.double(), (0, -cols % BLOCK)).reshape(rows, -1, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0))
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top > 0, e, 0.0).clamp(-111, 127)
    u = x * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(u / step) * step).view(rows, -1), e.squeeze(-1)


def _exact_values(pair):
    q, e = pair
    return (q.view(q.shape[0], -1, BLOCK) * torch.exp2(e).unsqueeze(-1)).view(q.shape[0], -1)


def _held(pair):
    q, s = pair
    return _exact_values((q.double(), s[:, :q.shape[0]].t().double() - 127))


def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op == 'quantize':
        x = s['x']
        got = [_nearest_blocks(x)] + ([_nearest_blocks(x.t())] if case['both'] else [])
        return [t for q, e in got for t in (q, None)]
    if op == 'dense':
        y = _exact_values(_nearest_blocks(s['x'])) @ _held(s['w']).t()
        y = y if s['bias'] is None else y + s['bias'].double()
        return y.clamp(min=0) if case['relu'] else y
    if op == 'product':
        return _held(s['a']) @ _held(s['b']).t()
    if op == 'linear':
        x, k, dy = s['x'].detach(), s['kernel'].detach(), s['dy']
        of = lambda t: _exact_values(_nearest_blocks(t))
        out = dict(y=of(x) @ of(k.t()).t(), dx=of(dy) @ of(k).t(), dkernel=of(x.t()) @ of(dy.t()).t())
        if s['bias'] is not None:
            out['y'] = out['y'] + s['bias'].detach().double()
            out['dbias'] = dy.double().sum(0)
        return out
    return _exact_adamw(s, case)


def _exact_adamw(s, case):
    """Parameter by parameter from the formulas; the states in 8 bits are decoded from their definition.  The new states in
    8 bits are random numbers' outcomes next to their borders and carry no value here."""
    b1, b2 = s['betas']
    e8 = case['states'] == '8bit'
    total = sum(g.double().square().sum() for g in s['grads'])
    norm = total.sqrt()
    factor = torch.clamp(case['clip'] / norm, max=1.0) if case['clip'] > 0 else 1.0
    params, ms, vs, at = [], torch.zeros(s['work'].numel(), dtype=torch.float64, device=DEV) if not e8 else None, None, 0
    vs = torch.zeros_like(ms) if ms is not None else None
    for p, g, wd in zip(s['params'], s['grads'], s['wd']):
        n = p.numel()
        span = slice(at, at + -(-n // BLOCK) * BLOCK)
        if e8:
            bl = slice(span.start // BLOCK, span.stop // BLOCK)
            m = (s['m'][span].double().view(-1, BLOCK) * torch.exp2(s['m_scale'][bl].double() - 127).view(-1, 1)).view(-1)[:n]
            c = s['v'][span].double().view(-1, BLOCK)
            v = (1 + (c % 8) / 8) * torch.exp2(torch.floor(c / 8) - 30 + s['v_scale'][bl].double().view(-1, 1) - 127)
            v = torch.where(c == 0, 0.0, v).view(-1)[:n]
        else:
            m, v = s['m'][span].double()[:n], s['v'][span].double()[:n]
        g = g.double().view(-1) * factor
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        q = p.double().view(-1)
        q = q - s['lr'] * wd * q - s['lr'] * (m / (1 - b1 ** 100)) / ((v / (1 - b2 ** 100)).sqrt() + s['eps'])
        params.append(q.view(p.shape))
        if not e8:
            ms[at:at + n], vs[at:at + n] = m, v
        at = span.stop
    out = dict(params=params, m=ms, v=vs, step=None)
    if e8:
        out.update(m_scale=None, v_scale=None)
    if case['clip'] > 0:
        out['norm'] = norm
    return out
