"""Work of the serving operators, as cases that can be timed and compared.

Four operators of one decoder layer that serves several requests at once:

* ``norm_fp8``: residual addition, RMS norm and e4m3 codes with one f32 scale
  for each 128 columns of a row (or the codes alone, without a norm);
* ``gemm_fp8``: the product that reads them, against weights with one f32
  scale for each block of 128 x 128;
* ``paged_append``: rotary positions applied to the new queries and keys, keys
  and values written to their slots of a paged cache;
* ``paged_attention``: one new token of each request over that cache.

Each case is a dict of plain values.  With ``own`` unset, ``run`` computes the
operators from elementary torch operations; with ``own`` set it makes the calls
of ``fluxvla_b200.ops``.  Both take what ``prepare`` gives.
"""
import math

import numpy as np
import torch

own = False

GROUP = 128                # columns that share a scale, rows too for weights
E4M3_MAX = 448.0
MIN_AMAX = 2.0 ** -60      # a group below this is coded against this
# scratch that a serving program keeps for paged_attention, zeroed once
WORKSPACE_BYTES = 64 << 20


def listed():
    return [
        # a single request decoding: its one token's residual row
        dict(name='norm one token', op='norm', rows=1, dim=2048,
             mode='gemma', x='f32', delta='bf16'),
        # action-expert rows of 64 requests, 51 each, modulated norm
        dict(name='norm expert rows', op='norm', rows=3264, dim=1024,
             mode='ada', x='bf16', delta='bf16'),
        # the MLP activations of an 848-row prompt before the down product
        dict(name='codes of mlp rows', op='norm', rows=848, dim=16384,
             mode='none', x='bf16', delta='none'),
        # query/key/value product of a single request's token
        dict(name='gemm qkv one token', op='gemm', m=1, n=2560, k=2048,
             epilogue='bf16'),
        # down product of 64 requests' tokens: a stream of weights
        dict(name='gemm down 64 tokens', op='gemm', m=64, n=2048, k=16384,
             epilogue='f32'),
        # a vision tower's second product over three views, ragged in K
        dict(name='gemm vision fc2', op='gemm', m=768, n=1152, k=4304,
             epilogue='bf16'),
        # gate and up of an 816-row prompt, gated GELU on the way out
        dict(name='gemm gate/up prompt', op='gemm', m=816, n=32768, k=2048,
             epilogue='geglu'),
        # one token of each of 64 requests
        dict(name='append 64 tokens', op='append', tokens=64, heads=8,
             kv_heads=1, dim=256, page=16, skipped=0.0, pairs='halves'),
        # 16 padded prompts of 816 rows, a fifth of the rows padding
        dict(name='append prompts', op='append', tokens=13056, heads=8,
             kv_heads=1, dim=256, page=48, skipped=0.2, pairs='halves'),
        # one request after its prompt and an action chunk
        dict(name='attend one request', op='attend', batch=1, heads=8,
             kv_heads=1, dim=256, page=16, shortest=867, longest=867),
        # 64 requests of very different lengths, one slot of them idle
        dict(name='attend 64 ragged', op='attend', batch=64, heads=8,
             kv_heads=1, dim=256, page=64, shortest=0, longest=8192),
        # grouped heads over long histories, pages of an odd size
        dict(name='attend long grouped', op='attend', batch=16, heads=32,
             kv_heads=4, dim=128, page=48, shortest=30000, longest=32768),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['norm', 'gemm', 'append', 'attend'])
    if op == 'norm':
        dim = _log(rng, 64, 16384)
        rows = max(1, min(_log(rng, 1, 32768), 848 * 16384 // dim))
        mode = rng.choice(['gemma', 'ada', 'rms', 'none'])
        return dict(op=op, rows=rows, dim=dim, mode=mode,
                    x=rng.choice(['f32', 'bf16']),
                    delta=rng.choice(['f32', 'bf16', 'none']))
    if op == 'gemm':
        n = 2 * _log(rng, 32, 16384)
        k = 16 * _log(rng, 8, 1024)
        m = max(1, min(_log(rng, 1, 4096), 816 * 32768 * 2048 // (n * k)))
        return dict(op=op, m=m, n=n, k=k,
                    epilogue=rng.choice(['bf16', 'f32', 'geglu']))
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    dim = rng.choice([64, 128, 256])
    page = rng.choice([8, 16, 32, 48, 64, 100, 128, 256])
    if op == 'append':
        tokens = _log(rng, 1, 13056)
        # not more elements than the largest listed case
        tokens = max(1, min(tokens, 13056 * 10 * 256 // ((group + 2) * kv * dim)))
        return dict(op=op, tokens=tokens, heads=kv * group, kv_heads=kv,
                    dim=dim, page=page, skipped=rng.choice([0.0, 0.1, 0.5]),
                    pairs=rng.choice(['halves', 'adjacent']))
    batch = _log(rng, 1, 256)
    longest = max(1, min(_log(rng, 1, 32768), (1 << 27) // (batch * kv * dim)))
    shortest = rng.choice([0, 1, longest // 2, longest])
    return dict(op=op, batch=batch, heads=kv * group, kv_heads=kv, dim=dim,
                page=page, shortest=min(shortest, longest), longest=longest)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
_TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16}


def _lengths(case):
    """Sequence lengths: spread evenly over the range, in a mixed order."""
    b, lo, hi = case['batch'], case['shortest'], case['longest']
    if b == 1:
        return [hi]
    step = next(s for s in (37, 41, 43, 47) if math.gcd(s, b) == 1)
    return [lo + (hi - lo) * ((i * step) % b) // (b - 1) for i in range(b)]


def _codes(x, rows_per_group):
    """e4m3 codes and scales of a matrix, for the products' inputs."""
    r, c = x.shape
    gr, gc = -(-r // rows_per_group), -(-c // GROUP)
    pad = torch.zeros(gr * rows_per_group, gc * GROUP, device=x.device)
    pad[:r, :c] = x
    blocks = pad.view(gr, rows_per_group, gc, GROUP)
    s = blocks.abs().amax(dim=(1, 3)).clamp(min=MIN_AMAX) / E4M3_MAX
    q = (blocks / s[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    q = q.view(gr * rows_per_group, gc * GROUP)[:r, :c].contiguous()
    return q.to(torch.float8_e4m3fn), s.contiguous()


def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, dt=torch.float32):
        return torch.randn(*shape, generator=g, device=dev).to(dt)

    s = dict(case)
    if case['op'] == 'norm':
        rows, dim = case['rows'], case['dim']
        dt = _TYPES[case['x']]
        # a few columns far larger than the rest, as in trained models
        col = 1 + 20 * (torch.rand(dim, generator=g, device=dev) > 0.99)
        s['x'] = (normal(rows, dim) * col).to(dt)
        s['delta'] = None
        if case['delta'] != 'none':
            s['delta'] = normal(rows, dim, dt=_TYPES[case['delta']])
            s['res'] = torch.empty_like(s['x'])
        s['w'] = s['mod'] = None
        if case['mode'] == 'gemma':
            s['w'] = (normal(dim) * 0.3).to(torch.bfloat16)
        elif case['mode'] == 'ada':
            s['mod'] = normal(2 * dim) * 0.3
        s['q'] = torch.empty(rows, dim, dtype=torch.float8_e4m3fn, device=dev)
        s['scales'] = torch.empty(rows, -(-dim // GROUP), device=dev)
    elif case['op'] == 'gemm':
        m, n, k = case['m'], case['n'], case['k']
        s['a'], s['a_scale'] = _codes(normal(m, k), 1)
        s['b'], s['b_scale'] = _codes(normal(n, k) * k ** -0.5, GROUP)
        out = n // 2 if case['epilogue'] == 'geglu' else n
        s['out'] = torch.empty(m, out, device=dev, dtype=torch.float32 if
                               case['epilogue'] == 'f32' else torch.bfloat16)
    elif case['op'] == 'append':
        t, h, kv, d = (case[x] for x in ('tokens', 'heads', 'kv_heads', 'dim'))
        page = case['page']
        pages = -(-t // page) + 3
        s['qkv'] = normal(t, (h + 2 * kv) * d, dt=torch.bfloat16)
        slots = torch.randperm(pages * page, generator=g, device=dev)[:t]
        skip = torch.rand(t, generator=g, device=dev) < case['skipped']
        s['slots'] = torch.where(skip, -1, slots).to(torch.int32)
        s['positions'] = torch.randint(0, 8192, (t,), generator=g, device=dev,
                                       dtype=torch.int32)
        s['k_cache'] = normal(pages, page, kv, d, dt=torch.bfloat16)
        s['v_cache'] = normal(pages, page, kv, d, dt=torch.bfloat16)
        inv = 10000.0 ** (-torch.arange(0, d, 2, device=dev).double() / d)
        ang = torch.arange(8192, device=dev).double()[:, None] * inv
        s['rope'] = torch.stack([ang.cos(), ang.sin()], -1).float()
        s['q_out'] = torch.empty(t, h, d, dtype=torch.bfloat16, device=dev)
    else:
        b, h, kv, d = (case[x] for x in ('batch', 'heads', 'kv_heads', 'dim'))
        page, lens = case['page'], _lengths(case)
        need = [-(-n // page) for n in lens]
        total, width = sum(need) + 2, max(1, -(-case['longest'] // page))
        perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
        table = torch.full((b, width), -1, dtype=torch.int32, device=dev)
        need_t = torch.tensor(need, device=dev)
        used = torch.arange(width, device=dev)[None] < need_t[:, None]
        table[used] = perm[:sum(need)]
        s['table'] = table
        s['lens'] = torch.tensor(lens, dtype=torch.int32, device=dev)
        s['q_in'] = normal(b, h, d, dt=torch.bfloat16)
        s['k_cache'] = normal(total, page, kv, d, dt=torch.bfloat16)
        s['v_cache'] = normal(total, page, kv, d, dt=torch.bfloat16)
        s['scale'] = 2.0 * d ** -0.5    # scores that spread, as trained ones
        s['out'] = torch.empty(b, h, d, dtype=torch.bfloat16, device=dev)
        s['lse'] = torch.empty(b, h, device=dev)
        s['workspace'] = torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8,
                                     device=dev)
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {'norm': _plain_norm, 'gemm': _plain_gemm, 'append': _plain_append,
            'attend': _plain_attend}[s['op']](s)


def _own(s):
    from fluxvla_b200 import _lib, ops
    if s['op'] == 'norm':
        mode = {'gemma': _lib.NORM_GEMMA_RMS, 'ada': _lib.NORM_ADA_RMS,
                'rms': _lib.NORM_RMS, 'none': _lib.NORM_NONE}[s['mode']]
        res = s.get('res')
        ops.norm_fp8(mode, s['x'], s['q'], s['scales'], delta=s['delta'],
                     res=res, w=s['w'], mod=s['mod'], eps=1e-6)
        return {'res': res, 'q': s['q'], 'scales': s['scales']}
    if s['op'] == 'gemm':
        epi = {'bf16': _lib.EPI_BF16, 'f32': _lib.EPI_F32_STORE,
               'geglu': _lib.EPI_GEGLU}[s['epilogue']]
        ops.gemm_fp8(s['a'], s['a_scale'], s['b'], s['b_scale'], s['out'],
                     epilogue=epi)
        return s['out']
    if s['op'] == 'append':
        q, k, v = _split(s)
        ops.paged_append(q, k, v, s['slots'], s['k_cache'], s['v_cache'],
                         q_out=s['q_out'], positions=s['positions'],
                         rope_cs=s['rope'],
                         rope_interleaved=s['pairs'] == 'adjacent')
        return {'q': s['q_out'], 'k_cache': s['k_cache'],
                'v_cache': s['v_cache']}
    ops.paged_attention(s['q_in'], s['k_cache'], s['v_cache'], s['table'],
                        s['lens'], s['out'], scale=s['scale'], lse=s['lse'],
                        workspace=s['workspace'])
    return {'out': s['out'], 'lse': s['lse']}


def _round_e4m3(t):
    """The e4m3 value nearest to each 64-bit value, ties to even."""
    a = t.abs().clamp(max=E4M3_MAX)
    e = torch.frexp(a.clamp(min=2.0 ** -6))[1] - 1
    step = torch.ldexp(torch.ones_like(a), e - 3)
    return (torch.round(a / step) * step * t.sign()).to(torch.float8_e4m3fn)


def _plain_norm(s):
    # 64 bits: a code is a whole step off where a value near the border
    # between two codes is computed less exactly
    x, dim = s['x'], s['dim']
    res = None
    if s['delta'] is not None:
        res = (x.double() + s['delta'].double()).to(x.dtype)
        x = res
    y = x.double()
    if s['mode'] != 'none':
        y = y * torch.rsqrt(y.square().mean(dim=1, keepdim=True) + 1e-6)
    if s['mode'] == 'gemma':
        y = y * (1.0 + s['w'].double())
    elif s['mode'] == 'ada':
        y = y * (1.0 + s['mod'][:dim].double()) + s['mod'][dim:].double()
    groups = -(-dim // GROUP)
    y = torch.nn.functional.pad(y, (0, groups * GROUP - dim))
    y = y.view(-1, groups, GROUP)
    scales = (y.abs().amax(dim=2).clamp(min=MIN_AMAX) / E4M3_MAX).float()
    t = (y / scales.double()[:, :, None]).view(-1, groups * GROUP)[:, :dim]
    return {'res': res, 'q': _round_e4m3(t), 'scales': scales}


def _spread(scale, rows, k, rows_per_group):
    full = scale.repeat_interleave(GROUP, 1)[:, :k]
    return full.repeat_interleave(rows_per_group, 0)[:rows]


def _plain_gemm(s):
    a = s['a'].float() * _spread(s['a_scale'], s['m'], s['k'], 1)
    b = s['b'].float() * _spread(s['b_scale'], s['n'], s['k'], GROUP)
    c = a @ b.t()
    if s['epilogue'] == 'geglu':
        # adjacent features are a gate and its up value
        gate, up = c[:, 0::2], c[:, 1::2]
        inner = 0.7978845608028654 * (gate + 0.044715 * gate * gate * gate)
        c = 0.5 * gate * (1 + torch.tanh(inner)) * up
    return c.to(s['out'].dtype)


def _split(s):
    t, h, kv, d = s['tokens'], s['heads'], s['kv_heads'], s['dim']
    rows = s['qkv'].view(t, h + 2 * kv, d)
    return rows[:, :h], rows[:, h:h + kv], rows[:, h + kv:]


def _rotate(x, cs, adjacent):
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    if adjacent:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _plain_append(s):
    q, k, v = _split(s)
    cs = s['rope'][s['positions'].long()]
    adjacent = s['pairs'] == 'adjacent'
    q = _rotate(q.float(), cs, adjacent).to(torch.bfloat16)
    k = _rotate(k.float(), cs, adjacent).to(torch.bfloat16)
    keep = s['slots'] >= 0
    at = s['slots'][keep].long()
    page = s['page']
    s['k_cache'][at // page, at % page] = k[keep]
    s['v_cache'][at // page, at % page] = v[keep]
    return {'q': q, 'k_cache': s['k_cache'], 'v_cache': s['v_cache']}


def _plain_attend(s):
    b, h, kv, d = s['batch'], s['heads'], s['kv_heads'], s['dim']
    n = s['longest']
    j = torch.arange(n, device=s['lens'].device)
    pages = s['table'].clamp(min=0).long()[:, j // s['page']]
    seen = j[None] < s['lens'][:, None]
    q = s['q_in'].float().view(b, kv, h // kv, d)
    k = s['k_cache'][pages, (j % s['page'])[None]].float()
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * s['scale']
    del k
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - top.clamp(min=-3e38))
    total = p.sum(dim=-1, keepdim=True)
    v = s['v_cache'][pages, (j % s['page'])[None]].float()
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / total.clamp(min=1e-30)
    lse = (top + torch.log(total)).view(b, h)
    return {'out': out.view(b, h, d).to(torch.bfloat16), 'lse': lse}


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    if case['op'] == 'norm':
        n = case['rows'] * case['dim']
        size = {'f32': 4, 'bf16': 2, 'none': 0}
        moved = size[case['x']] + 1 + size[case['delta']]
        if case['delta'] != 'none':
            moved += size[case['x']]
        groups = case['rows'] * -(-case['dim'] // GROUP)
        weights = {'gemma': 2, 'ada': 8}.get(case['mode'], 0) * case['dim']
        return {'bytes': n * moved + 4 * groups + weights, 'flops': 8 * n}
    if case['op'] == 'gemm':
        m, n, k = case['m'], case['n'], case['k']
        groups = -(-k // GROUP)
        out = m * n * {'bf16': 2, 'f32': 4, 'geglu': 1}[case['epilogue']]
        return {'bytes': (m + n) * k + out + 4 * groups * (m - -n // GROUP),
                'flops': 2 * m * n * k}
    if case['op'] == 'append':
        t, h, kv, d = (case[x] for x in ('tokens', 'heads', 'kv_heads', 'dim'))
        kept = int(t * (1 - case['skipped']))
        table = min(t, 8192) * d * 4
        return {'bytes': (t * h + 2 * kept * kv) * d * 4 + 8 * t + table,
                'flops': 3 * (t * h + kept * kv) * d}
    lens = _lengths(case)
    total, b = sum(lens), case['batch']
    return {'bytes': total * case['kv_heads'] * case['dim'] * 4 +
            b * case['heads'] * (case['dim'] * 4 + 4) + 4 * b +
            4 * sum(-(-n // case['page']) for n in lens),
            'flops': 4 * total * case['heads'] * case['dim']}


# --------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {'norm': _exact_norm, 'gemm': _exact_gemm, 'append': _exact_append,
            'attend': _exact_attend}[case['op']](s)


def _e4m3_values():
    """All finite values of the format that are not negative, in order."""
    low = np.arange(8) * 2.0 ** -9
    high = [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)]
    return np.concatenate([low, np.array(high)[:-1]])    # the last is NaN


def _exact_norm(s):
    h = s['x'].double()
    res = None
    if s['delta'] is not None:
        # the residual as it is stored is what the norm is taken of
        res = h + s['delta'].double()
        h = res.to(s['x'].dtype).double()
    rows, dim = h.shape
    if s['mode'] != 'none':
        h = h / torch.sqrt((h * h).sum(1, keepdim=True) / dim + 1e-6)
    if s['mode'] == 'gemma':
        h = h + h * s['w'].double()
    elif s['mode'] == 'ada':
        scale, shift = s['mod'].double().split(dim)
        h = h + h * scale + shift
    values = torch.from_numpy(_e4m3_values()).to(h.device)
    borders = (values[1:] + values[:-1]) / 2
    q = torch.empty_like(h)
    scales = torch.empty(rows, -(-dim // GROUP), dtype=torch.float64,
                         device=h.device)
    for i, c in enumerate(range(0, dim, GROUP)):
        part = h[:, c:c + GROUP]
        top = torch.maximum(part.abs().amax(1), torch.full_like(h[:, 0], MIN_AMAX))
        scales[:, i] = top / E4M3_MAX
        # codes are relative to the scale that is stored, in 32 bits
        t = part / scales[:, i:i + 1].float().double()
        a = t.abs()
        # on a border the even code wins: the lower one if its place is even
        lo = torch.bucketize(a, borders)
        up = torch.bucketize(a, borders, right=True)
        at = torch.where(lo % 2 == 0, lo, up)
        q[:, c:c + GROUP] = values[at] * torch.sign(t)
    return {'res': res, 'q': q, 'scales': scales}


def _exact_gemm(s):
    m, n, k = s['m'], s['n'], s['k']
    c = torch.zeros(m, n, dtype=torch.float64, device=s['a'].device)
    rows = s['b_scale'].double().repeat_interleave(GROUP, 0)[:n]
    for i, at in enumerate(range(0, k, GROUP)):
        part = s['a'][:, at:at + GROUP].double() @ s['b'][:, at:at + GROUP].double().t()
        c += part * s['a_scale'][:, i:i + 1].double() * rows[:, i]
    if s['epilogue'] == 'geglu':
        x, up = c.view(m, n // 2, 2).unbind(-1)
        z = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
        c = x / (1 + torch.exp(-2 * z)) * up
    return c


def _exact_append(s):
    t, h, kv, d = s['tokens'], s['heads'], s['kv_heads'], s['dim']
    rows = s['qkv'].double().view(t, h + 2 * kv, d)
    cs = s['rope'].double()[s['positions'].long()]
    turn = torch.complex(cs[..., 0], cs[..., 1])[:, None]
    turned = rows[:, :h + kv]
    if s['pairs'] == 'adjacent':
        z = torch.complex(turned[..., 0::2].contiguous(),
                          turned[..., 1::2].contiguous()) * turn
        turned = torch.view_as_real(z).reshape(t, h + kv, d)
    else:
        half = d // 2
        z = torch.complex(turned[..., :half].contiguous(),
                          turned[..., half:].contiguous()) * turn
        turned = torch.cat([z.real, z.imag], -1)
    keep = torch.nonzero(s['slots'] >= 0)[:, 0]
    at = s['slots'][keep].long()
    kc = s['k_cache'].double().flatten(0, 1)
    vc = s['v_cache'].double().flatten(0, 1)
    kc[at], vc[at] = turned[keep, h:], rows[keep, h + kv:]
    shape = s['k_cache'].shape
    return {'q': turned[:, :h].contiguous(), 'k_cache': kc.view(shape),
            'v_cache': vc.view(shape)}


def _exact_attend(s):
    b, h, kv, d = s['batch'], s['heads'], s['kv_heads'], s['dim']
    out = torch.zeros(b, h, d, dtype=torch.float64, device=s['lens'].device)
    lse = torch.full((b, h), -math.inf, dtype=torch.float64, device=out.device)
    for i, n in enumerate(_lengths(s)):
        if n == 0:
            continue
        pages = s['table'][i, :-(-n // s['page'])].long()
        k = s['k_cache'][pages].flatten(0, 1)[:n].double()
        v = s['v_cache'][pages].flatten(0, 1)[:n].double()
        q = s['q_in'][i].double().view(kv, h // kv, d)
        score = torch.einsum('cgd,ncd->cgn', q, k) * s['scale']
        lse[i] = torch.logsumexp(score, -1).view(h)
        out[i] = torch.einsum('cgn,ncd->cgd', torch.softmax(score, -1),
                              v).reshape(h, d)
    return {'out': out, 'lse': lse}
