"""Rotary positions (`rotary.rotary_tables`, `rotary.rotary_embedding`) against their definition in 64 bits."""
import math

import pytest
import torch

import oracle.serving_ref as S

pytestmark = pytest.mark.gpu
H, F = torch.float16, torch.float32


@pytest.fixture(scope="module")
def rotary():
    from ascend910a_extras import rotary as r

    return r


def _check_tables(got, want, amp):
    # the angle in turns is rounded to 32 bits (half a step of at most 1/2 turn: 3.2 * 2^-24 rad), sine and cosine are
    # good to 2 steps (4 * 2^-24), the factor and the rounding to fp32 cost half a step each; fp16 rounds once more
    for g, w in zip(got, want):
        tol = 10 * 2.0 ** -24 * amp
        if g.dtype == H:
            tol = tol + w.abs() * 2.0 ** -11 + 2.0 ** -25
        assert ((g.cpu().double() - w).abs() <= tol).all(), float((g.cpu().double() - w).abs().max())


def _check_rotated(got, x, pos, cos, sin, interleaved):
    # two products and a sum in fp32 (three half steps of the sum of magnitudes), one rounding to fp16
    want = S.rotary_embedding_ref(x, pos, cos, sin, interleaved)
    size = S.rotary_embedding_ref(x.abs(), pos, cos.abs(), -sin.abs(), interleaved).abs()
    size = torch.maximum(size, S.rotary_embedding_ref(x.abs(), pos, cos.abs(), sin.abs(), interleaved).abs())
    tol = want.abs() * 2.0 ** -11 + 2.0 ** -25 + size * 3 * 2.0 ** -24
    assert got.dtype == H and got.is_contiguous() and got.shape == x.shape
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any(), int(bad.sum())
    r = 2 * cos.shape[1]
    assert torch.equal(got.cpu()[..., r:], x[..., r:])


SCALINGS = [
    dict(),
    dict(scaling="linear", factor=4.0),
    dict(scaling="ntk", factor=8.0),
    dict(scaling="dynamic", factor=2.0, original=300),
    dict(scaling="dynamic", factor=2.0, original=5000),     # not stretched yet
    dict(scaling="yarn", factor=8.0, original=256),
    dict(scaling="yarn", factor=4.0, original=64, beta_fast=16.0, beta_slow=2.0),
    dict(scaling="wavelength", factor=8.0, original=512, low=1.0, high=4.0),
    dict(scaling="yarn", factor=4.0, original=4),  # no pair turns even once: all but the first are divided
]


@pytest.mark.parametrize("dtype", [H, F])
@pytest.mark.parametrize("kw", SCALINGS, ids=lambda k: "-".join(str(v) for v in k.values()) or "plain")
@pytest.mark.parametrize("positions,dim,base", [(1000, 64, 10000.0), (1, 128, 500000.0), (17, 20, 10000.0), (40, 600, 1e6)])
def test_tables(rotary, dev, kw, positions, dim, base, dtype):
    freqs, amp = S.rotary_frequencies_ref(dim, base, positions, **kw)
    names = {"original": "original_max_position", "low": "low_freq_factor", "high": "high_freq_factor"}
    got = rotary.rotary_tables(positions, dim, base, dtype=dtype, device=dev, **{names.get(k, k): v for k, v in kw.items()})
    assert got[0].shape == (positions, dim // 2) and got[0].dtype == dtype
    _check_tables(got, S.rotary_tables_ref(positions, freqs, amp), amp)


def test_tables_with_a_factor_per_pair(rotary, dev):
    factors = torch.linspace(1, 30, 48)
    freqs, amp = S.rotary_frequencies_ref(96, 10000.0, 700, "pairs", 32.0, 4096, pair_factors=factors)
    got = rotary.rotary_tables(700, 96, scaling="pairs", factor=32.0, original_max_position=4096,
                               pair_factors=factors.to(dev), dtype=F)
    _check_tables(got, S.rotary_tables_ref(700, freqs, amp), amp)
    got = rotary.rotary_tables(700, 96, scaling="pairs", pair_factors=factors.to(dev), attention_factor=1.5, dtype=F)
    _check_tables(got, S.rotary_tables_ref(700, freqs, 1.5), 1.5)


def test_tables_keep_their_accuracy_at_far_positions(rotary, dev):
    n = 2_000_001
    cos, sin = rotary.rotary_tables(n, 4, 1e4, dtype=F, device=dev)
    freqs, _ = S.rotary_frequencies_ref(4, 1e4, n)
    want = S.rotary_tables_ref(n, freqs, 1.0)
    # the reference itself rounds the angle in 64 bits: 2e6 * 2^-53 rad, nothing beside 2^-24
    _check_tables((cos, sin), want, 1.0)


def test_tables_feed_the_neox_operator(rotary, ops, dev):
    cos, sin = rotary.rotary_tables(300, 64, device=dev)
    q, k = torch.randn(9, 4, 64).half().to(dev), torch.randn(9, 2, 64).half().to(dev)
    pos = torch.arange(9, dtype=torch.int32, device=dev) * 31
    for a, b in zip(ops.rope(q, k, pos, cos, sin), rotary.rotary_embedding(q, k, pos, cos, sin)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [H, F])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,d,r", [(1, 1, 1, 8, 2), (5, 4, 2, 64, 64), (33, 32, 8, 128, 64), (7, 3, 1, 80, 20),
                                              (3, 5, 5, 96, 94), (65, 2, 1, 256, 256), (2, 1, 0, 72, 48), (2, 0, 3, 24, 16)])
def test_embedding(rotary, dev, tokens, hq, hk, d, r, interleaved, dtype):
    g = torch.Generator().manual_seed(tokens * 7 + r)
    q, k = torch.randn(tokens, hq, d, generator=g).half(), torch.randn(tokens, hk, d, generator=g).half()
    cos, sin = (t.to(dtype) for t in S.rotary_tables_ref(77, S.rotary_frequencies_ref(r, 1e4, 77)[0], 1.25))
    pos = torch.randint(0, 77, (tokens,), generator=g, dtype=torch.int32)
    oq, ok = rotary.rotary_embedding(*(t.to(dev) for t in (q, k, pos, cos, sin)), interleaved=interleaved)
    _check_rotated(oq, q, pos, cos, sin, interleaved)
    _check_rotated(ok, k, pos, cos, sin, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_embedding_reads_views(rotary, dev, interleaved):
    """q, k inside a fused projection, heads with something in front of the rotated part, one head for all tokens,
    one token for all rows; positions outside the tables."""
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(19, (6 + 2 + 2) * 64, generator=g).half().to(dev)
    q, k, _ = qkv.split([6 * 64, 2 * 64, 2 * 64], 1)
    q, k = q.unflatten(1, (6, 64)), k.unflatten(1, (2, 64))
    cos, sin = (t.half() for t in S.rotary_tables_ref(40, S.rotary_frequencies_ref(32, 1e4, 40)[0], 1.0))
    pos = torch.randint(-3, 45, (19,), generator=g, dtype=torch.int32)
    args = [t.to(dev) for t in (pos, cos, sin)]
    for x in rotary.rotary_embedding(q, k, *args, interleaved=interleaved):
        _check_rotated(x, (q if x.size(1) == 6 else k).cpu(), pos, cos, sin, interleaved)
    wide = torch.randn(19, 6, 192, generator=g).half().to(dev)
    tail = wide[..., 128:]
    shared = torch.randn(19, 1, 64, generator=g).half().to(dev).expand(19, 5, 64)
    same = torch.randn(1, 3, 64, generator=g).half().to(dev).expand(19, 3, 64)
    for a, b in ((tail, shared), (same, tail)):
        for x, y in zip(rotary.rotary_embedding(a, b, *args, interleaved=interleaved), (a, b)):
            _check_rotated(x, y.cpu(), pos, cos, sin, interleaved)
    for x, y in zip(rotary.rotary_embedding(tail.transpose(0, 1)[:, :6], wide.transpose(0, 1)[:, :6, 64:128], args[0][:6], *args[1:],
                                            interleaved=interleaved), (tail, wide[..., 64:128])):
        _check_rotated(x, y.transpose(0, 1)[:, :6].cpu(), pos[:6], cos, sin, interleaved)


def test_nothing_to_rotate(rotary, dev):
    q = torch.zeros(0, 4, 64, dtype=H, device=dev)
    cos = torch.zeros(3, 32, dtype=H, device=dev)
    oq, ok = rotary.rotary_embedding(q, q[:, :2], torch.zeros(0, dtype=torch.int32, device=dev), cos, cos)
    assert oq.shape == (0, 4, 64) and ok.shape == (0, 2, 64)
    assert rotary.rotary_tables(0, 64, device=dev)[0].shape == (0, 32)


def test_infinities_and_nan_stay_in_their_pairs(rotary, dev):
    q = torch.randn(4, 2, 64).half()
    q[0, 0, 3], q[1, 1, 40], q[2, 0, 63] = math.inf, math.nan, -math.inf
    cos, sin = (t.half() for t in S.rotary_tables_ref(9, S.rotary_frequencies_ref(48, 1e4, 9)[0], 1.0))
    pos = torch.tensor([0, 3, 8, 1], dtype=torch.int32)
    for interleaved in (False, True):
        got = rotary.rotary_embedding(*(t.to(dev) for t in (q, q, pos, cos, sin)), interleaved=interleaved)[0].cpu()
        want = S.rotary_embedding_ref(q, pos, cos, sin, interleaved)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        ok = want.isfinite()
        assert torch.allclose(got.double()[ok], want[ok], rtol=2.0 ** -10, atol=2.0 ** -20)


def test_types_and_devices_are_checked(rotary, dev):
    q, k = (torch.zeros(4, n, 64, dtype=H, device=dev) for n in (2, 1))
    pos, c = torch.zeros(4, dtype=torch.int32, device=dev), torch.zeros(9, 32, dtype=H, device=dev)
    for args, match in [((q, k, pos.long(), c, c), "int32"), ((q, k, pos, c, c.float()), "float16"),
                        ((q, k, pos, c.double(), c.double()), "float16"), ((q, k.bfloat16(), pos, c, c), "float16"),
                        ((q, k, pos.cpu(), c, c), "GPU device"), ((q, k, pos, c.cpu(), c), "GPU device"),
                        ((torch.zeros(4, 3, 68, dtype=H, device=dev)[:, :, 4:], k, pos, c, c), "multiples of 8"),
                        ((torch.zeros(4 * 2 * 64 + 4, dtype=H, device=dev)[4:].view(4, 2, 64), k, pos, c, c), "aligned"),
                        ((q, k, pos, torch.zeros(9 * 32 + 1, dtype=H, device=dev)[1:].view(9, 32), c), "aligned")]:
        with pytest.raises(RuntimeError, match=match):
            rotary.rotary_embedding(*args)
    with pytest.raises(RuntimeError, match="float32"):
        rotary.rotary_tables(4, 64, scaling="pairs", pair_factors=torch.ones(32, dtype=H, device=dev))
    with pytest.raises(RuntimeError, match="rotary_dim/2"):
        rotary.rotary_tables(4, 64, scaling="pairs", pair_factors=torch.ones(31, device=dev))
    with pytest.raises(RuntimeError, match="invalid argument"):
        rotary.rotary_tables(4, 64, base=-1.0, device=dev)


def test_in_a_graph_and_on_another_stream(rotary, dev):
    q, k = torch.randn(40, 4, 64).half().to(dev), torch.randn(40, 2, 64).half().to(dev)
    pos = torch.arange(40, dtype=torch.int32, device=dev)

    def step():
        cos, sin = rotary.rotary_tables(300, 48, scaling="dynamic", factor=2.0, original_max_position=100, device=dev)
        return [cos, sin, *rotary.rotary_embedding(q, k, pos, cos, sin), *rotary.rotary_embedding(q, k, pos, cos, sin, interleaved=True)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        q.copy_(torch.randn(40, 4, 64).half())
        pos.add_(60)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), i
