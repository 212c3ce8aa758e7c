"""64-bit restatements of the serving operators, for their tests."""
import math

import torch

F64 = torch.float64
GROUP = 128


def e4m3_grid():
    """The finite e4m3 values that are not negative, in order of their codes."""
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).to(F64)


def to_e4m3(t):
    """Nearest e4m3 value of 64-bit values, ties to the even code, saturating."""
    g = e4m3_grid().to(t.device)
    a = t.abs().clamp(max=448.0)
    hi = torch.searchsorted(g, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - g[lo], g[hi] - a
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.where(t < 0, -g[pick], g[pick])


def norm_fp8(mode, x, delta=None, w=None, mod=None, eps=1e-6):
    """(res, codes as values, scales f32)."""
    from fluxvla_b200 import _lib
    h = x
    if delta is not None:
        h = (x.to(F64) + delta.to(F64)).to(x.dtype)
    y = h.to(F64)
    rows, dim = y.shape
    if mode != _lib.NORM_NONE:
        y = y / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
    if mode == _lib.NORM_GEMMA_RMS:
        y = y * (1 + w.to(F64))
    elif mode == _lib.NORM_ADA_RMS:
        y = y * (1 + mod[:dim].to(F64)) + mod[dim:].to(F64)
    groups = -(-dim // GROUP)
    q = torch.empty_like(y)
    s = torch.empty(rows, groups, device=x.device)
    for i in range(groups):
        part = y[:, i * GROUP:(i + 1) * GROUP]
        top = part.abs().nan_to_num(0.0, posinf=math.inf).amax(1)
        s[:, i] = (top.clamp(min=2.0 ** -60) / 448.0).float()
        q[:, i * GROUP:(i + 1) * GROUP] = to_e4m3(part / s[:, i:i + 1].to(F64))
    return h, q, s


def gemm_fp8(a, sa, b, sb):
    """(product, sum of the terms' magnitudes), both 64-bit."""
    m, k = a.shape
    n = b.shape[0]
    c = torch.zeros(m, n, dtype=F64, device=a.device)
    mag = torch.zeros_like(c)
    rows = sb.to(F64).repeat_interleave(GROUP, 0)[:n]
    for i in range(sa.shape[1]):
        x = a[:, i * GROUP:(i + 1) * GROUP].to(F64)
        y = b[:, i * GROUP:(i + 1) * GROUP].to(F64).t()
        s = sa[:, i:i + 1].to(F64) * rows[:, i]
        c += s * (x @ y)
        mag += s.abs() * (x.abs() @ y.abs())
    return c, mag


def gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) *
                                     (x + 0.044715 * x ** 3)))


def rotate(x, positions, rope, interleaved):
    c = rope.to(F64)[positions.long()][:, None]
    x = x.to(F64)
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
    else:
        a, b = x.chunk(2, -1)
    u, v = a * c[..., 0] - b * c[..., 1], b * c[..., 0] + a * c[..., 1]
    if interleaved:
        return torch.stack([u, v], -1).flatten(-2)
    return torch.cat([u, v], -1)


def attention(q, kc, vc, table, lens, scale):
    """(out, lse, sum of p * |v|, largest sum of |q||k| * scale) per head."""
    bsz, heads, dim = q.shape
    page, kv = kc.shape[1], kc.shape[2]
    g = heads // kv
    out = torch.zeros(bsz, heads, dim, dtype=F64, device=q.device)
    mag = torch.zeros_like(out)
    lse = torch.full((bsz, heads), -math.inf, dtype=F64, device=q.device)
    qk = torch.zeros(bsz, heads, dtype=F64, device=q.device)
    for b in range(bsz):
        n = int(lens[b])
        if n <= 0:
            continue
        pages = table[b, :-(-n // page)].long()
        k = kc[pages].flatten(0, 1)[:n].to(F64)
        v = vc[pages].flatten(0, 1)[:n].to(F64)
        x = q[b].to(F64).view(kv, g, dim)
        s = torch.einsum('cgd,ncd->cgn', x, k) * scale
        p = torch.softmax(s, -1)
        out[b] = torch.einsum('cgn,ncd->cgd', p, v).reshape(heads, dim)
        mag[b] = torch.einsum('cgn,ncd->cgd', p, v.abs()).reshape(heads, dim)
        lse[b] = torch.logsumexp(s, -1).reshape(heads)
        qk[b] = (torch.einsum('cgd,ncd->cgn', x.abs(), k.abs()).amax(-1) *
                 abs(scale)).reshape(heads)
    return out, lse, mag, qk
