"""The 8-bit linear layer with a scale per block of 128, its gradients, and the clipping of gradients by their global norm: what is timed.

Each case is one pass through one operator, in two forms: the plain one (`own` false: elementary torch operations in 32 bits) and the
framework's kernels (`own` true: autolabel_amd.fp8 and autolabel_amd.clip as a program calls them).

The 8-bit format.  A row is cut into blocks of 128 values along the contracted axis (the last block may be short).  A block is stored as
8-bit floating point values q (e4m3: 4 exponent bits, 3 of mantissa, largest 448; e5m2: 5 and 2, largest 57344) and ONE power of two:
    s = the smallest power of two >= 2^-126 with max |x| / s <= largest value of the type   (1 for a block of zeros)
    q = x / s rounded to the nearest value of the type, ties to even
The division is exact, so q is one rounding of x and every implementation gets the same q.
"""
import math

import torch

own = False

DTYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
F8 = {'e4m3': (torch.float8_e4m3fn, 8), 'e5m2': (torch.float8_e5m2, 15)}     # the type, the exponent of its largest value
BLOCK = 128


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    lin = lambda name, m, k, n, dtype, relu: {'name': name, 'op': 'linear', 'm': m, 'k': k, 'n': n, 'dtype': dtype, 'relu': relu}
    back = lambda name, m, k, n, dtype, gfmt: {'name': name, 'op': 'backward', 'm': m, 'k': k, 'n': n, 'dtype': dtype, 'gfmt': gfmt}
    clip = lambda name, sizes, dtype, clipped, out: {'name': name, 'op': 'clip', 'sizes': sizes, 'dtype': dtype, 'clipped': clipped, 'out': out}
    return [
        # one point asked for its 512 features (a click in the viewer): one row through a layer of the wide feature head, latency
        lin('linear one point', 1, 512, 512, 'fp16', True),
        # the composited hidden activation of a 4096-ray batch through the head's last layer
        lin('linear rays', 4096, 512, 512, 'fp16', False),
        # 3-D queries come in batches of 50000 points, which is no multiple of any tile
        lin('linear points', 50000, 512, 512, 'fp16', True),
        # every sample of a 4096-ray batch, 256 a ray, through a hidden layer of the head: streams 2 GB
        lin('linear samples', 1 << 20, 512, 512, 'fp16', True),
        # the class head's first layer: 512 features and 16 geometry features in, 64 out: a short last block
        lin('linear classes', 65537, 528, 64, 'bf16', True),
        # a generic square layer with its rows in the thousands: bound by the matrix cores
        lin('linear square', 8192, 4096, 4096, 'bf16', False),
        # the compression autoencoder's first layer on the rows of one feature map, 480 x 360 at half size, gradients in e5m2
        back('backward map', 43200, 512, 128, 'fp16', 'e5m2'),
        # odd in every direction: smaller than a block in K, ragged in M and N
        back('backward ragged', 1003, 77, 130, 'bf16', 'e4m3'),
        # the wide head's hidden layer in a training step on half a batch's samples: a contraction over 524288 rows
        back('backward samples', 1 << 19, 512, 512, 'fp16', 'e4m3'),
        # the field's own parameter blocks: the hash table of 16 levels (most of its gradient is zero) and the four heads, the semantic ones 512 wide
        clip('clip field', '14229504,24576,22528,532480,34816', 'fp32', True, True),
        # a step that needs no clipping, in place: the gradients are only read
        clip('clip idle', '14229504,24576,22528,532480,34816', 'fp32', False, False),
        # the layers of a small network, weights and odd biases, gradients in 16 bits
        clip('clip layers', ','.join('65536,512,%d,%d' % (32768 + 7 * i, 1 + 13 * i) for i in range(14)), 'bf16', True, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(['linear', 'linear', 'backward', 'clip'])
    if op == 'clip':
        count, total = rng.randint(1, 60), _log_int(rng, 64, 14 << 20)
        cut = [rng.random() ** 3 + 1e-3 for _ in range(count)]
        sizes = [max(1, int(total * c / sum(cut))) for c in cut]
        return {'op': op, 'sizes': ','.join(map(str, sizes)), 'dtype': rng.choice(['fp32', 'fp16', 'bf16']), 'clipped': (c := rng.random() < 0.7), 'out': c}
    k, n = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
    # rows up to a million, and no more work or data than a layer of the wide head (backward: half of that) or the square layer has
    top = min(1 << 20, (1 << 30) // (k + n), (1 << 37) // (k * n)) // (2 if op == 'backward' else 1)
    m = _log_int(rng, 1, top)
    case = {'op': op, 'm': m, 'k': k, 'n': n, 'dtype': rng.choice(['fp16', 'bf16'])}
    return {**case, 'relu': rng.random() < 0.5} if op == 'linear' else {**case, 'gfmt': rng.choice(['e4m3', 'e5m2'])}


# --------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _activations(g, m, k, dtype):
    """Rows of a hidden layer: about half of the values 0 (behind a ReLU), rows of different sizes, a few columns that stand out."""
    x = torch.randn(m, k, generator=g, device='cuda', dtype=torch.float16)
    x.clamp_(min=0)
    x.mul_(torch.rand(m, 1, generator=g, device='cuda').mul_(2).add_(0.05).half())
    x.mul_(torch.rand(1, k, generator=g, device='cuda').lt_(0.02).mul_(7).add_(1).half())
    return x.to(dtype)


def _weights(g, n, k):
    return (torch.rand(n, k, generator=g, device='cuda') * 2 - 1) * math.sqrt(6.0 / (n + k))


def prepare(case, seed):
    g = _gen(seed)
    if case['op'] == 'clip':
        dtype = DTYPES[case['dtype']]
        grads = []
        for n in map(int, case['sizes'].split(',')):
            t = torch.randn(n, generator=g, device='cuda') * 1e-2
            if n > (1 << 20):     # a hash table's gradient: most entries were not touched by the batch
                t *= torch.rand(n, generator=g, device='cuda') < 0.3
            grads.append(t.to(dtype))
        norm = math.sqrt(sum(float(t.float().square().sum(dtype=torch.float64)) for t in grads))
        return {'case': case, 'grads': grads, 'max_norm': (0.37 if case['clipped'] else 1.9) * norm + 1e-4,
                'out': [torch.empty_like(t) for t in grads] if case['out'] else None}
    m, k, n, dtype = case['m'], case['k'], case['n'], DTYPES[case['dtype']]
    x = _activations(g, m, k, dtype)
    w = _weights(g, n, k)
    if case['op'] == 'linear':     # the layer's weights, laid out once: blocks along K
        q, e = _blocks(w, 'e4m3')
        return {'case': case, 'x': x, 'w': _held(q, e, k, 'e4m3')}
    gy = (torch.randn(m, n, generator=g, device='cuda', dtype=torch.float16) * 0.05).to(dtype)
    gy.mul_(torch.rand(m, 1, generator=g, device='cuda').to(dtype))
    q, e = _blocks(w.t().contiguous(), 'e4m3')      # the transposed weights, for the data gradient: blocks along N
    return {'case': case, 'x': x, 'g': gy, 'wt': _held(q, e, n, 'e4m3')}


def _held(q, e, cols, fmt):
    """The blocks as they are held: 8-bit values [rows, blocks * 128] (zeros behind the last column), and the powers of two as exponent + 127."""
    rows, nb = e.shape
    scale = torch.full((rows, (nb + 3) // 4 * 4), 127, dtype=torch.uint8, device=q.device)
    scale[:, :nb] = (e + 127).to(torch.uint8)
    return {'q': q.reshape(rows, nb * BLOCK).to(F8[fmt][0]), 'scale': scale, 'cols': cols, 'fmt': fmt}


# ----------------------------------------------------------------------------------------------------------- plain forms
def _pow2(e):
    """2^e for whole e in [-126, 127], from its bits (a device's exp2 may be a rounding off, and that would move ties)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _blocks(x, fmt):
    """q [rows, blocks, 128] as 32-bit values of the 8-bit type, and the exponents e [rows, blocks] of the powers of two."""
    rows, cols = x.shape
    nb = (cols + BLOCK - 1) // BLOCK
    b = x.float()
    if nb * BLOCK != cols:
        b = torch.cat([b, b.new_zeros(rows, nb * BLOCK - cols)], 1)
    b = b.reshape(rows, nb, BLOCK)
    f, e = torch.frexp(b.abs().amax(-1))                    # max = f 2^e with f in [1/2, 1): 2 f 2^(e - 1)
    e = e - 1 - F8[fmt][1] + (f > 0.875).to(e.dtype)        # both types' largest value is 1.75 2^emax
    e = torch.where(f == 0, torch.zeros_like(e), e).clamp(min=-126)
    return (b * _pow2(-e)[..., None]).to(F8[fmt][0]).float(), e


def _values(q, e):
    """The values that the blocks stand for, [rows, blocks * 128] in 32 bits."""
    return (q * _pow2(e)[..., None]).reshape(q.shape[0], -1)


def _held_values(w):
    return _values(w['q'].float().reshape(w['q'].shape[0], -1, BLOCK), w['scale'][:, :w['q'].shape[1] // BLOCK].int() - 127)


def _linear(s):
    y = _values(*_blocks(s['x'], 'e4m3')) @ _held_values(s['w']).t()
    return (y.clamp(min=0) if s['case']['relu'] else y).to(s['x'].dtype)


def _backward(s):
    c = s['case']
    dx = _values(*_blocks(s['g'], c['gfmt'])) @ _held_values(s['wt']).t()
    gt, xt = _values(*_blocks(s['g'].t(), c['gfmt'])), _values(*_blocks(s['x'].t(), 'e4m3'))     # blocks along the rows
    # a long contraction: 32-bit products of up to 4096 rows each, their sums in 64 bits
    step = BLOCK * min(32, gt.shape[1] // BLOCK)
    pad = -gt.shape[1] % step
    gt, xt = (torch.cat([t, t.new_zeros(t.shape[0], pad)], 1).reshape(t.shape[0], -1, step) for t in (gt, xt))
    dw = torch.bmm(gt.transpose(0, 1).contiguous(), xt.permute(1, 2, 0).contiguous()).sum(0, dtype=torch.float64)
    return {'dx': dx.to(s['x'].dtype), 'dw': dw.float()}


def _clip(s):
    norm = torch.stack([t.float().square().sum(dtype=torch.float64) for t in s['grads']]).sum().sqrt().float()
    factor = (s['max_norm'] / (norm + 1e-6)).clamp(max=1.0)
    return [norm] + [t.copy_(t.float() * factor) if s['out'] is None else o.copy_(t.float() * factor) for t, o in zip(s['grads'], s['out'] or s['grads'])]


# ----------------------------------------------------------------------------------------------------------------- passes
def run(s):
    op = s['case']['op']
    if own:
        from autolabel_amd import clip, fp8
        if op == 'clip':
            norm = clip.clip_grad_norm_(s['grads'], s['max_norm'], out=s['out'])
            return [norm] + (s['grads'] if s['out'] is None else s['out'])
        if op == 'linear':
            return fp8.linear(s['x'], fp8.Fp8Blocks(**s['w']), relu=s['case']['relu'])
        dx, dw = fp8.linear_backward(s['g'], s['x'], fp8.Fp8Blocks(**s['wt']), grad_fmt=s['case']['gfmt'])
        return {'dx': dx, 'dw': dw}
    return {'linear': _linear, 'backward': _backward, 'clip': _clip}[op](s)


def work(case):
    if case['op'] == 'clip':
        n = sum(map(int, case['sizes'].split(',')))
        return {'bytes': n * torch.empty((), dtype=DTYPES[case['dtype']]).element_size() * (2 if case['out'] else 1), 'flops': 3 * n}
    m, k, n = case['m'], case['k'], case['n']
    nb = lambda c: (c + BLOCK - 1) // BLOCK
    if case['op'] == 'linear':
        return {'bytes': 2 * m * (k + n) + n * k + n * nb(k), 'flops': 2 * m * k * n}
    return {'bytes': 2 * m * (n + k) + n * k + k * nb(n) + 2 * m * k + 4 * n * k, 'flops': 4 * m * k * n}


# ------------------------------------------------------------------------------------------------- the definition, 64 bits
def _two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_blocks(x, fmt):
    """What the blocks of the rows of x stand for, from the format's definition, in 64 bits: [rows, cols]."""
    digits, lowest, largest = {'e4m3': (3, -6, 448.0), 'e5m2': (2, -14, 57344.0)}[fmt]
    x = x.double()
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], BLOCK):
        b = x[:, at:at + BLOCK]
        most = b.abs().max(1, keepdim=True).values
        s = _two_to(torch.ceil(torch.log2(most.clamp(min=1e-300) / largest)).clamp(min=-126.0))
        s = torch.where(most / s > largest, 2 * s, s)                            # log2 may be a rounding off at a power of two
        s = torch.where((most / (s / 2) <= largest) & (s > 2.0 ** -126), s / 2, s)
        s = torch.where(most == 0, torch.ones_like(s), s)
        v = b / s
        exp = torch.frexp(v)[1] - 1                                              # |v| in [2^exp, 2^(exp + 1))
        step = _two_to(exp.clamp(min=lowest) - digits)
        out[:, at:at + BLOCK] = torch.round(v / step) * step * s                 # torch.round: ties to even
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'clip':
        g = [t.double() for t in s['grads']]
        norm = torch.sqrt(sum((t * t).sum() for t in g))
        factor = min(1.0, s['max_norm'] / (float(norm) + 1e-6))
        return [norm] + [t * factor for t in g]
    if case['op'] == 'linear':
        w = s['w']['q'].double() * _two_to(s['w']['scale'].int() - 127).repeat_interleave(BLOCK, 1)[:, :s['w']['q'].shape[1]]
        w = w[:, :case['k']]
        y = _exact_blocks(s['x'], 'e4m3') @ w.t()
        return torch.where(y > 0, y, torch.zeros_like(y)) if case['relu'] else y
    wt = s['wt']['q'].double() * _two_to(s['wt']['scale'].int() - 127).repeat_interleave(BLOCK, 1)[:, :s['wt']['q'].shape[1]]
    wt = wt[:, :case['n']]
    dx = _exact_blocks(s['g'], case['gfmt']) @ wt.t()
    dw = _exact_blocks(s['g'].t().contiguous(), case['gfmt']) @ _exact_blocks(s['x'].t().contiguous(), 'e4m3').t()
    return {'dx': dx, 'dw': dw}
