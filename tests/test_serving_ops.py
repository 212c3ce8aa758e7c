"""What the serving operators refuse, and the weight codes, without a GPU."""
import ctypes as C

import pytest
import torch

from fluxvla_b200 import _lib, ops, pack
from tests import serving_ref as R


def refused(fn, args, text, code=_lib.FVB_ERR_INVALID_ARG):
    L = _lib.lib()
    rc = getattr(L, fn)(C.byref(args), None)
    assert rc == code, (rc, L.fvb_last_error())
    assert text in L.fvb_last_error().decode()


def with_(args, **kw):
    out = type(args)()
    C.memmove(C.byref(out), C.byref(args), C.sizeof(args))
    for k, v in kw.items():
        setattr(out, k, v)
    return out


P = 4096     # an aligned address; nothing here reaches a launch


def norm_args():
    return _lib.NormFp8Args(mode=_lib.NORM_RMS, rows=2, dim=256, x=P, ld_x=256,
                            eps=1e-6, q=P, ld_q=256, scales=P, ld_scales=2)


@pytest.mark.parametrize('kw,text,code', [
    (dict(rows=-1), 'bad shape', 1), (dict(dim=0), 'bad shape', 1),
    (dict(mode=_lib.NORM_LAYER), 'bad mode', 1), (dict(mode=6), 'bad mode', 1),
    (dict(dim=16385, ld_x=16385, ld_q=16385, ld_scales=129), 'over 16384', 2),
    (dict(mode=_lib.NORM_NONE, dim=2 ** 31 - 1, ld_x=2 ** 31, ld_q=2 ** 31,
          ld_scales=2 ** 24), 'over 134215680', 2),
    (dict(x=None), 'NULL', 1), (dict(q=None), 'NULL', 1),
    (dict(scales=None), 'NULL', 1),
    (dict(mode=_lib.NORM_GEMMA_RMS), 'weight required', 1),
    (dict(mode=_lib.NORM_ADA_RMS), 'modulation required', 1),
    (dict(delta=P, ld_delta=256), 'come together', 1),
    (dict(res=P, ld_res=256), 'come together', 1),
    (dict(ld_x=255), 'stride', 1), (dict(ld_q=255), 'stride', 1),
    (dict(ld_scales=1), 'stride', 1),
    (dict(delta=P, ld_delta=255, res=P, ld_res=256), 'stride', 1),
    (dict(eps=-1.0), 'eps', 1), (dict(eps=float('nan')), 'eps', 1)])
def test_norm_fp8_refusals(kw, text, code):
    refused('fvb_norm_fp8', with_(norm_args(), **kw), text, code)


def gemm_args():
    return _lib.GemmFp8Args(a=P, lda=256, a_scale=P, ld_as=2, b=P, ldb=256,
                            b_scale=P, ld_bs=2, m=4, n=128, k=256, epilogue=0,
                            out=P, ldo=128)


@pytest.mark.parametrize('kw,text', [
    (dict(m=-1), 'bad shape'), (dict(n=0), 'bad shape'),
    (dict(k=0), 'bad shape'), (dict(epilogue=2), 'bad epilogue'),
    (dict(epilogue=4), 'bad epilogue'),
    (dict(epilogue=3, n=127), 'even feature'),
    (dict(a=None), 'NULL'), (dict(b_scale=None), 'NULL'),
    (dict(out=None), 'NULL'), (dict(lda=255), 'stride'),
    (dict(ldb=128), 'stride'), (dict(ld_as=1), 'stride'),
    (dict(ld_bs=1), 'stride'), (dict(ldo=127), 'stride'),
    (dict(a=P + 8), '16B aligned'), (dict(lda=264), '16B aligned'),
    (dict(b=P + 1), '16B aligned')])
def test_gemm_fp8_refusals(kw, text):
    refused('fvb_gemm_fp8', with_(gemm_args(), **kw), text)


@pytest.mark.parametrize('kw', [
    dict(m=2 ** 31 - 1), dict(n=2 ** 31 - 1, ldo=2 ** 31),
    dict(k=2 ** 31 - 1, lda=2 ** 31, ldb=2 ** 31, ld_as=2 ** 24,
         ld_bs=2 ** 24)])
def test_gemm_fp8_sizes_at_the_end_of_32_bits(kw):
    refused('fvb_gemm_fp8', with_(gemm_args(), **kw), 'too large',
            _lib.FVB_ERR_UNSUPPORTED)


def append_args():
    return _lib.PagedAppendArgs(
        q=P, k=P, v=P, q_out=P, k_cache=P, v_cache=P, n_pages=4, page_size=16,
        slots=P, positions=P, rope_cs=P, max_pos=10, tokens=3, heads=2,
        kv_heads=1, head_dim=64)


@pytest.mark.parametrize('kw,text', [
    (dict(tokens=-1), 'bad shape'), (dict(kv_heads=0), 'bad shape'),
    (dict(head_dim=63), 'bad shape'), (dict(heads=-1), 'bad shape'),
    (dict(page_size=0), 'cache shape'), (dict(n_pages=-1), 'cache shape'),
    (dict(k=None), 'NULL'), (dict(slots=None), 'NULL'),
    (dict(v_cache=None), 'NULL'), (dict(q=None), 'q and q_out'),
    (dict(q_out=None), 'q and q_out'), (dict(positions=None), 'positions'),
    (dict(max_pos=0), 'positions'), (dict(rope_cs=P + 4), 'positions')])
def test_paged_append_refusals(kw, text):
    refused('fvb_paged_append', with_(append_args(), **kw), text)


def attn_args():
    return _lib.PagedAttnArgs(
        q=P, q_row_stride=128, q_head_stride=64, k_cache=P, kc_page_stride=1024,
        kc_row_stride=64, kc_head_stride=64, v_cache=P, vc_page_stride=1024,
        vc_row_stride=64, vc_head_stride=64, n_pages=4, page_size=16,
        page_table=P, ld_table=4, max_pages=4, seq_lens=P, out=P,
        out_row_stride=128, out_head_stride=64, batch=2, heads=2, kv_heads=1,
        head_dim=64, scale=1.0, workspace=P, workspace_bytes=1 << 30)


@pytest.mark.parametrize('kw,text,code', [
    (dict(batch=-1), 'bad batch', 1), (dict(heads=0), 'bad batch', 1),
    (dict(heads=3, kv_heads=2), 'bad batch', 1),
    (dict(kv_heads=0), 'bad batch', 1), (dict(head_dim=72), 'head_dim 72', 2),
    (dict(q=None), 'NULL', 1), (dict(seq_lens=None), 'NULL', 1),
    (dict(page_table=None), 'NULL', 1), (dict(page_size=0), 'cache shape', 1),
    (dict(ld_table=3), 'cache shape', 1), (dict(n_pages=-1), 'cache shape', 1),
    (dict(max_pages=1 << 27, ld_table=1 << 27), 'keys a sequence', 2),
    (dict(k_cache=P + 8), '16B aligned', 1),
    (dict(vc_row_stride=68), '16B aligned', 1),
    (dict(q=P + 2), '4-byte', 1), (dict(out_head_stride=66), '8-byte', 1),
    (dict(workspace=None), 'workspace needs', 5),
    (dict(workspace_bytes=100), 'workspace needs', 5),
    (dict(workspace=P + 8), 'workspace needs', 5)])
def test_paged_attention_refusals(kw, text, code):
    refused('fvb_paged_attention', with_(attn_args(), **kw), text, code)


@pytest.mark.parametrize('page,pages', [
    (48, 44739241), (8, 2 ** 28 - 9), (16, 2 ** 27 - 3), (1, 2 ** 31 - 128),
    (1, 2 ** 31 - 1), (256, 2 ** 23 - 20)])
def test_paged_attention_tables_at_the_end_of_32_bits(page, pages):
    """Lengths that the kernel could not round up to whole units."""
    refused('fvb_paged_attention',
            with_(attn_args(), batch=1, page_size=page, max_pages=pages,
                  ld_table=pages), 'keys a sequence', _lib.FVB_ERR_UNSUPPORTED)


@pytest.mark.parametrize('kw', [
    dict(batch=2 ** 31 - 1, max_pages=0), dict(batch=2 ** 31 - 300, max_pages=7),
    dict(batch=2 ** 30, max_pages=16), dict(batch=2 ** 28, heads=8, kv_heads=8)])
def test_paged_attention_batches_at_the_end_of_32_bits(kw):
    refused('fvb_paged_attention', with_(attn_args(), ld_table=16, **kw),
            'sequences of up to', _lib.FVB_ERR_UNSUPPORTED)


def test_paged_attention_heads_at_the_end_of_32_bits():
    refused('fvb_paged_attention',
            with_(attn_args(), batch=1, heads=2 ** 25, head_dim=64),
            'heads', _lib.FVB_ERR_UNSUPPORTED)


def test_workspace_does_not_depend_on_batch():
    L = _lib.lib()
    sizes = set()
    for batch in (1, 64, 100000):
        sizes.add(L.fvb_paged_attention_workspace_bytes(
            C.byref(with_(attn_args(), batch=batch))))
    assert len(sizes) == 1 and sizes.pop() > 4096
    assert ops.paged_attention_workspace_bytes(8, 1, 256) > 0
    with pytest.raises(_lib.FVBError, match='head_dim 72'):
        ops.paged_attention_workspace_bytes(8, 1, 72)


def test_null_argument_structures():
    L = _lib.lib()
    for fn in ('fvb_norm_fp8', 'fvb_gemm_fp8', 'fvb_paged_append',
               'fvb_paged_attention'):
        assert getattr(L, fn)(None, None) == _lib.FVB_ERR_INVALID_ARG
    assert L.fvb_paged_attention_workspace_bytes(None) == -1


def test_empty_calls_do_nothing():
    L = _lib.lib()
    for fn, a in (('fvb_norm_fp8', with_(norm_args(), rows=0)),
                  ('fvb_gemm_fp8', with_(gemm_args(), m=0)),
                  ('fvb_paged_append', with_(append_args(), tokens=0)),
                  ('fvb_paged_attention', with_(attn_args(), batch=0))):
        assert getattr(L, fn)(C.byref(a), None) == 0, L.fvb_last_error()


def test_tensors_on_the_host_are_refused():
    e = torch.zeros(2, 128, dtype=torch.float8_e4m3fn)
    s = torch.zeros(2, 1)
    x = torch.zeros(2, 128)
    with pytest.raises(ValueError, match='must be a CUDA tensor'):
        ops.norm_fp8(_lib.NORM_RMS, x, e, s)
    with pytest.raises(ValueError, match='expected float32 or bfloat16'):
        ops.norm_fp8(_lib.NORM_RMS, x.half(), e, s)
    with pytest.raises(ValueError, match='must be a CUDA tensor'):
        ops.gemm_fp8(e, s, e, s[:1], x)
    k = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    c = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match='must be a CUDA tensor'):
        ops.paged_append(None, k, k, i, c, c)
    with pytest.raises(ValueError, match='must be a CUDA tensor'):
        ops.paged_attention(k, c, c, i[:, None], i, k, scale=1.0, workspace=s)


@pytest.mark.parametrize('n,k', [(1, 1), (128, 128), (130, 300), (256, 144)])
def test_quantize_blocks(n, k):
    g = torch.Generator().manual_seed(n + k)
    w = torch.randn(n, k, generator=g)
    w[0] = 0
    q, s = pack.quantize_blocks(w)
    assert q.dtype == torch.float8_e4m3fn and q.shape == w.shape
    assert s.shape == (-(-n // 128), -(-k // 128))
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            b = w[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].double()
            top = b.abs().max().clamp(min=2.0 ** -60) / 448
            assert s[i, j] == top.float()
            got = q[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].double()
            # half a step of e4m3 (relative 2^-4, or of the smallest step)
            t = b / s[i, j].double()
            assert ((got - t).abs() <= t.abs() * 2.0 ** -4 + 2.0 ** -10).all()


def test_reference_rounding_matches_the_type():
    """The tests' own e4m3 rounding, on values that 32 bits hold."""
    t = torch.cat([torch.linspace(-460, 460, 20001), torch.linspace(-.05, .05, 20001)])
    want = t.clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert torch.equal(R.to_e4m3(t.double()), want)
