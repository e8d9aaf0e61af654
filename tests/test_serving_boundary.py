"""Refusals of the operators around the paged caches, without a GPU: the Python layer raises RuntimeError, the C ABI
returns its codes before it touches the device."""
import ctypes

import pytest
import torch

import cabi

H, I = torch.float16, torch.int32


def _raises(fn, *args, match=None, **kw):
    with pytest.raises(RuntimeError, match=match):
        fn(*args, **kw)


def _half(*shape):
    return torch.zeros(*shape, dtype=H)


def _int(*shape):
    return torch.zeros(*shape, dtype=I)


def test_rotary_embedding_refusals():
    from ascend910a_extras.rotary import rotary_embedding as f

    q, k, pos, c = _half(4, 2, 64), _half(4, 1, 64), _int(4), _half(9, 32)
    _raises(f, q[0], k, pos, c, c, match="3D")
    _raises(f, q, k[:3], pos, c, c, match="match q")
    _raises(f, q, k[..., :32], pos, c, c, match="match q")
    _raises(f, q, k, pos[:3], c, c, match="one entry per token")
    _raises(f, _half(4, 2, 60), _half(4, 1, 60), pos, _half(9, 30), _half(9, 30), match="multiple of 8")
    _raises(f, q, k, pos, _half(9, 33), _half(9, 33), match="rotary_dim")
    _raises(f, q, k, pos, c, _half(8, 32), match="rotary_dim")
    _raises(f, q, k, pos, _half(9, 0), _half(9, 0), match="rotary_dim")
    _raises(f, q, k, pos, _half(0, 32), _half(0, 32), match="rows")
    _raises(f, q, k, pos, _half(9, 64)[:, ::2], c, match="contiguous")
    _raises(f, _half(4, 64, 2).transpose(1, 2), k, pos, c, c, match="next to each other")
    _raises(f, _half(4, 2, 68)[..., :64], k, pos, c, c, match="multiples of 8")
    _raises(f, q.float(), k, pos, c, c, match="float16")
    _raises(f, q, k, pos, c, c, match="GPU device")


def test_rotary_tables_refusals():
    from ascend910a_extras.rotary import rotary_tables as f

    _raises(f, 8, 64, scaling="other", match="scaling")
    _raises(f, 8, 64, dtype=torch.bfloat16, match="dtype")
    _raises(f, 8, 64, attention_factor=0.0, match="attention_factor")
    _raises(f, 8, 64, scaling="pairs", match="pair_factors")
    _raises(f, 8, 64, pair_factors=torch.ones(32), match="pair_factors")
    _raises(f, 8, 63, match="even")
    _raises(f, -1, 64, match="negative")
    _raises(f, 8, 64, device="cpu", match="GPU device")


def test_c_abi_rotary():
    lib = cabi.lib()
    p = ctypes.c_void_p(16)

    def tables(n=8, r=64, base=1e4, scaling=0, factor=1.0, orig=0.0, low=1.0, high=4.0, amp=0.0, pairs=None, out=p):
        return lib.aops_rotary_tables(out, out, 0, n, r, base, scaling, factor, orig, low, high, amp, pairs, None)

    assert tables(n=0) == 0
    assert tables(out=None) == -1
    for bad in (dict(n=-1), dict(r=0), dict(r=3), dict(base=0.0), dict(base=float("nan")), dict(base=float("inf")),
                dict(factor=0.0), dict(factor=float("nan")), dict(amp=-1.0), dict(amp=float("nan")), dict(scaling=7),
                dict(scaling=-1), dict(scaling=2, r=2), dict(scaling=3), dict(scaling=4), dict(scaling=5),
                dict(scaling=4, orig=64.0, low=0.0), dict(scaling=4, orig=64.0, low=32.0, high=1.0, base=1.0),
                dict(scaling=4, orig=64.0, low=1.0, high=32.0), dict(scaling=4, orig=64.0, low=32.0, high=1.0, base=0.5),
                dict(n=1 << 30, r=65536), dict(scaling=5, orig=64.0, low=4.0, high=4.0), dict(scaling=6), dict(scaling=6, factor=2.0, pairs=p),
                dict(scaling=6, factor=2.0, orig=1.0, pairs=p), dict(n=1 << 31)):
        assert tables(**bad) == -1, bad

    def embed(tokens=0, hq=2, hk=1, d=64, r=64, n=9, s=(128, 64, 64, 64), ptr=p):
        return lib.aops_rotary_f16(ptr, ptr, ptr, ptr, ptr, 0, ptr, ptr, tokens, hq, hk, d, r, n, 0, *s, None)

    assert embed() == 0 and embed(n=0) == 0 and embed(tokens=5, hq=0, hk=0) == 0
    for bad in (dict(tokens=-1), dict(hq=-1), dict(d=0), dict(d=60), dict(r=0), dict(r=66), dict(r=7), dict(n=-1),
                dict(s=(4, 64, 64, 64)), dict(s=(128, -64, 64, 64)), dict(tokens=4, n=0), dict(tokens=4, ptr=None),
                dict(tokens=1 << 31), dict(tokens=1 << 30, hq=32), dict(tokens=1, hq=(1 << 63) - 1),
                dict(tokens=1, hk=(1 << 63) - 1)):
        assert embed(**bad) == -1, bad


def test_page_refusals():
    from ascend910a_extras import paged

    kc = [_half(8, 4, 16, 16) for _ in range(2)]
    t, l, c, i = _int(3, 4), _int(3), _int(8), _int(2)
    _raises(paged.copy_pages, [], [], i, i, match="at least one cache")
    _raises(paged.copy_pages, kc, [_half(8, 4, 8, 16)], i, i, match="same shape|GPU device")
    _raises(paged.copy_pages, [_half(8, 4, 16)], [], i, i, match="num_blocks")
    _raises(paged.copy_pages, [_half(8, 4, 16, 8)], [], i, i, match="num_blocks")
    _raises(paged.copy_pages, [_half(8, 4, 16, 32)[..., ::2]], [], i, i, match="contiguous")
    _raises(paged.copy_pages, [kc[0].float()], [], i, i, match="float16")
    _raises(paged.copy_pages, kc, kc, i, i, match="GPU device")
    _raises(paged.fork_sequences, t, l, i, c, kc, kc, match="GPU device")
    _raises(paged.compact_pages, t, l, c, kc, kc, match="GPU device")
    _raises(paged.extend_sequences, t, l, l, c, 16, match="GPU device")
    _raises(paged.extend_sequences, t[0], l, l, c, 16, match="2D")
    _raises(paged.free_sequences, t, l, i, c, 16, match="GPU device")
    _raises(paged.free_sequences, t, l[:, None], i, c, 16, match="1D|GPU device")


def test_c_abi_pages():
    lib = cabi.lib()
    p = ctypes.c_void_p(16)
    many = (ctypes.c_void_p * 257)(*([16] * 257))
    holes = (ctypes.c_void_p * 2)(16, None)
    assert lib.aops_pages_workspace(5, 100) == 4 * (4 + 100 + 200)
    assert lib.aops_pages_workspace(500, 100) == 4 * (4 + 100 + 500)
    assert lib.aops_pages_workspace(-1, 100) == 0 and lib.aops_pages_workspace(1, 1 << 31) == 0

    def copy(caches=many, n=2, pairs=0, blocks=8, row=64, block=16, ptr=p):
        return lib.aops_copy_pages_f16(caches, n, ptr, ptr, pairs, blocks, row, block, None)

    assert copy() == 0 and copy(blocks=0, pairs=3) == 0
    for bad in (dict(n=0), dict(n=257), dict(pairs=-1), dict(blocks=-1), dict(row=0), dict(row=40), dict(block=0),
                dict(pairs=2, caches=None), dict(pairs=2, caches=holes), dict(pairs=2, ptr=None),
                dict(row=1 << 20, block=1 << 20), dict(pairs=1 << 31), dict(pairs=1 << 24), dict(pairs=(1 << 63) - 1)):
        assert copy(**bad) == -1, bad

    def fork(caches=many, n=2, seqs=3, width=4, children=2, blocks=8, row=64, block=16, ptr=p, ws=p, ws_bytes=1 << 20):
        return lib.aops_fork_sequences_f16(ptr, ptr, seqs, width, ptr, children, ptr, blocks, caches, n, row, block, ptr,
                                           ptr, ptr, ws, ws_bytes, None)

    for bad in (dict(n=0), dict(n=257), dict(seqs=-1), dict(width=-1), dict(children=-1), dict(blocks=-1), dict(row=8),
                dict(block=0), dict(ptr=None), dict(caches=None), dict(caches=holes), dict(children=(1 << 24) - 1),
                dict(children=(1 << 63) - 1)):
        assert fork(**bad) == -1, bad
    assert fork(ws=None) == -2 and fork(ws_bytes=lib.aops_pages_workspace(2, 8) - 1) == -2
    assert fork(children=0, blocks=0) == 0

    def compact(caches=many, n=2, seqs=3, width=4, blocks=8, row=64, block=16, ptr=p, ws=p, ws_bytes=1 << 20):
        return lib.aops_compact_pages_f16(ptr, ptr, seqs, width, ptr, blocks, caches, n, row, block, ptr, ptr, ptr, ws,
                                          ws_bytes, None)

    for bad in (dict(n=0), dict(seqs=-1), dict(width=-1), dict(blocks=-1), dict(row=8), dict(block=0), dict(ptr=None),
                dict(caches=holes)):
        assert compact(**bad) == -1, bad
    assert compact(ws=None) == -2 and compact(ws_bytes=lib.aops_pages_workspace(0, 8) - 1) == -2

    def extend(seqs=3, width=4, block=16, blocks=8, ptr=p, ws=p, ws_bytes=1 << 20):
        return lib.aops_extend_sequences(ptr, ptr, ptr, seqs, width, block, ptr, blocks, ptr, ptr, ptr, ws, ws_bytes, None)

    for bad in (dict(seqs=-1), dict(width=-1), dict(block=0), dict(blocks=-1), dict(ptr=None), dict(seqs=(1 << 24) - 1)):
        assert extend(**bad) == -1, bad
    assert extend(ws=None) == -2 and extend(ws_bytes=lib.aops_pages_workspace(3, 8) - 1) == -2
    assert extend(seqs=0, blocks=0) == 0

    def free(seqs=3, width=4, block=16, rows=2, blocks=8, ptr=p):
        return lib.aops_free_sequences(ptr, ptr, seqs, width, block, ptr, rows, ptr, blocks, ptr, None)

    for bad in (dict(seqs=-1), dict(width=-1), dict(block=0), dict(rows=-1), dict(blocks=-1), dict(ptr=None),
                dict(rows=1 << 24)):
        assert free(**bad) == -1, bad
    assert free(blocks=0) == 0


def test_chunk_attention_refusals():
    from ascend910a_extras.paged import paged_attention_chunk as f

    q, c, t, l, s = _half(3, 4, 64), _half(8, 8, 16, 16), _int(2, 4), _int(2), _int(3)
    _raises(f, q[0], c, c, t, l, s, match="3D")
    _raises(f, q.transpose(0, 1), c, c, t, l, s, match="contiguous")
    _raises(f, q, _half(8, 8, 16, 8), _half(8, 8, 16, 8), t, l, s, match="16")
    _raises(f, q, c, c[:4], t, l, s, match="same shape")
    _raises(f, _half(3, 4, 72), c, c, t, l, s, match="head_dim")
    _raises(f, _half(3, 4, 272), c, c, t, l, s, match="head_dim")
    _raises(f, _half(3, 4, 48), c, c, t, l, s, match="whole heads")
    _raises(f, _half(3, 5, 64), c, c, t, l, s, match="num_kv_heads")
    _raises(f, q, c, c, t, _int(3), s, match="context_lens")
    _raises(f, q, c, c, t, l, l, match="query_starts")
    _raises(f, q, c, c, t, l, s, scale=-1.0, match="scale")
    _raises(f, q, c, c, t, l, s, scale=float("inf"), match="scale")
    _raises(f, q, c, c, t, l, s, window=-1, match="window")
    _raises(f, q, c, c, t, l, s, match="GPU device")


def test_c_abi_chunk_attention():
    lib = cabi.lib()
    p = ctypes.c_void_p(16)

    def run(tokens=4, seqs=2, hq=4, hk=2, d=64, block=16, pages=4, blocks=8, scale=0.1, window=0, ptr=p, ws=p, ws_bytes=1 << 30):
        return lib.aops_paged_attention_chunk_f16(ptr, ptr, ptr, ptr, ptr, ptr, ptr, None, scale, window, ws, ws_bytes, tokens,
                                                  seqs, hq, hk, d, block, pages, blocks, None)

    assert run(tokens=0) == 0 and run(seqs=0) == 0
    for bad in (dict(tokens=-1), dict(seqs=-1), dict(hq=0), dict(hk=0), dict(hq=5), dict(d=0), dict(d=72), dict(d=272),
                dict(block=0), dict(pages=-1), dict(blocks=-1), dict(scale=0.0), dict(scale=float("nan")), dict(window=-1),
                dict(ptr=None), dict(tokens=1 << 30, hq=4, hk=1), dict(tokens=1 << 31), dict(block=1 << 20, pages=1 << 20),
                dict(tokens=1 << 22, seqs=1 << 22)):
        assert run(**bad) == -1, bad
    assert run(ws=None) == -2
    size = lib.aops_paged_attention_chunk_workspace
    # short tables: no partial results; long ones: two slots per share, rows of the largest tile, and the plan
    assert size(4, 2, 4, 2, 64, 16, 4) == 16
    assert size(4, 2, 4, 2, 64, 16, 400) == 2 * 2 * 128 * 16 * 66 * 4 + (4 + 3 * 3 + 1 + 128) * 4
    assert size(100000, 1, 2, 1, 128, 1 << 16, 32767) == 16  # the partition counts in 32 bits
    assert run(pages=400, ws_bytes=size(4, 2, 4, 2, 64, 16, 400) - 1) == -2
    assert size(4, 2, 5, 2, 64, 16, 4) == 0 and size(4, 2, 4, 2, 24, 16, 4) == 0


def test_c_abi_pages_refuse_rows_that_pass_32_bits():
    """A workgroup counts the columns of a row in 32 bits, in steps of its threads: the last step must not wrap."""
    lib = cabi.lib()
    p = ctypes.c_void_p(16)
    many = (ctypes.c_void_p * 2)(16, 16)
    for width in (0x7fffff01, 0x7fffffff):
        assert lib.aops_fork_sequences_f16(p, p, 1, width, p, 1, p, 8, many, 2, 64, 16, p, p, p, p, 1 << 20, None) == -1
        assert lib.aops_extend_sequences(p, p, p, 1, width, 16, p, 8, p, p, p, p, 1 << 20, None) == -1
        assert lib.aops_free_sequences(p, p, 1, width, 16, p, 1, p, 8, p, None) == -1
        assert lib.aops_compact_pages_f16(p, p, 1, width, p, 8, many, 2, 64, 16, p, p, p, p, 1 << 20, None) == -1


def test_chunk_attention_refuses_scales_that_leave_fp32():
    """With 2^56 the scores of any finite queries and keys can be told from a masked place; beyond that rows could come out
    as if they saw nothing."""
    from ascend910a_extras.paged import paged_attention_chunk as f

    lib, p = cabi.lib(), ctypes.c_void_p(16)
    for scale in (2.0 ** 57, 1e27, 3e38):
        assert lib.aops_paged_attention_chunk_f16(p, p, p, p, p, p, p, None, scale, 0, p, 1 << 30, 4, 2, 4, 2, 64, 16, 4, 8, None) == -1
        _raises(f, _half(3, 4, 64), _half(8, 8, 16, 16), _half(8, 8, 16, 16), _int(2, 4), _int(2), _int(3), scale=scale, match="2\\^56")
