"""Attention of a chunk of new tokens over the paged caches (`paged.paged_attention_chunk`) against its definition in
64 bits."""
import math

import pytest
import torch

import oracle.ops_ref as R
import oracle.serving_ref as S

pytestmark = pytest.mark.gpu
H, I = torch.float16, torch.int32


@pytest.fixture(scope="module")
def paged():
    from ascend910a_extras import paged as p

    return p


def _case(new, ctx, hq, hkv, d, block, seed=0, extra_pages=1, spread=1.0):
    """Random caches with a shuffled table; the pages' places behind a context hold NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-n // block)) for n in ctx]
    width = max(need + [1]) + extra_pages
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=g)
    tables = torch.full((len(ctx), width), pool + 7, dtype=I)  # entries behind the context are no pages
    k = torch.randn(pool, block, hkv, d, generator=g) * spread
    v = torch.randn(pool, block, hkv, d, generator=g)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at:at + n].int()
        if ctx[b] > 0 and ctx[b] % block:
            k[order[at + n - 1], ctx[b] % block:] = math.nan
            v[order[at + n - 1], ctx[b] % block:] = math.inf
        at += n
    k[order[at:]], v[order[at:]] = math.nan, math.nan
    starts = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=I)
    q = (torch.randn(int(starts[-1]), hq, d, generator=g) * spread).half()
    return q, R.nz_pack(k.half()), R.nz_pack(v.half()), tables, torch.tensor(ctx, dtype=I), starts


def _tolerances(case, o, lse, scale, window, ref):
    """Bounds from the roundings there are: a score is exact products added in fp32 (D + 1 half steps of its size at
    most) and scaled (one), the exponential is good to 2^-22 of itself and its argument to half a step (2^-24) of the largest
    scaled score; a weight for the product is rounded to fp16 (2^-11 of itself, 2^-25 * 2^-6 of the row's largest
    below that), sums in fp32 cost another half step per 32 keys, and the result is rounded to fp16 once."""
    q, kc, vc, tables, ctx, starts = case
    d = q.shape[-1]
    finite = lambda t: torch.where(t.isfinite(), t.double().abs(), torch.zeros((), dtype=torch.float64))  # noqa: E731
    s = (finite(q).max() * finite(kc).max() * d * scale).item()
    per_score = min(s, 60.0) * (d + 4) * 2.0 ** -24 * 1.5
    keys = int(ctx.max())
    weight = 2.0 ** -11 + 2.0 ** -21 + 2 * per_score + (keys / 32 + 8) * 2.0 ** -23 + keys * 2.0 ** -31
    # sum of weight * |v| is at most the largest |v|, and on average as much smaller as the result itself
    return ref[0].abs() * (2.0 ** -11 + weight) + weight * finite(vc).max().item() + 2.0 ** -24, \
        per_score + 2.0 ** -20 + ref[1].abs() * 2.0 ** -22


def _check(paged, dev, case, scale=None, window=0):
    q, kc, vc, tables, ctx, starts = case
    ref = S.paged_attention_chunk_ref(*case, scale=scale, window=window)
    o, lse = paged.paged_attention_chunk(*(t.to(dev) for t in case), scale=scale, window=window, return_lse=True)
    o, lse = o.cpu().double(), lse.cpu().double()
    tol_o, tol_l = _tolerances(case, o, lse, scale or q.shape[-1] ** -0.5, window, ref)
    covered = torch.zeros(q.shape[0], dtype=torch.bool)
    for b in range(len(ctx)):
        covered[int(starts[b]):int(starts[b + 1])] = True
    # a row that sees a NaN of the cache is NaN, one that sees nothing is 0 and -inf
    o, lse, ref = o[covered], lse[covered], (ref[0][covered], ref[1][covered])
    tol_o, tol_l = tol_o[covered], tol_l[covered]
    seen, nothing = ref[1].isfinite(), ref[1] == -math.inf
    assert torch.equal(lse.isnan(), ref[1].isnan()) and torch.equal(lse == -math.inf, nothing)
    assert (o[nothing] == 0).all() and torch.equal(o.isnan(), ref[0].isnan())
    o, lse, ref, tol_o, tol_l = o[seen], lse[seen], (ref[0][seen], ref[1][seen]), tol_o[seen], tol_l[seen]
    err = (o - ref[0]).abs()
    assert (err <= tol_o).all(), (float((err / tol_o).max()), float(err.max()))
    # over all values the errors average out: half a step of the result, half a step of each weight, three times over
    assert err.norm() <= 3 * 2.0 ** -11 * ref[0].norm() + 1e-12, float(err.norm() / ref[0].norm())
    el = (lse - ref[1]).abs()
    assert (el <= tol_l).all(), float((el / tol_l).max())


SMALL = [
    # new tokens, context lengths, query heads, kv heads, head_dim, block size
    ([1], [1], 1, 1, 128, 16),
    ([1, 1, 1], [5, 33, 300], 8, 2, 128, 16),
    ([5, 2, 4], [5, 70, 600], 8, 2, 128, 128),
    ([3, 1, 0, 7], [10, 64, 40, 7], 4, 4, 64, 32),
    ([17, 1, 40], [17, 257, 256], 6, 2, 80, 16),
    ([33], [90], 8, 8, 128, 16),            # one row too many for the stream path
    ([32], [90], 8, 8, 128, 16),
    ([70, 9], [70, 530], 16, 4, 128, 64),
    ([129, 64], [200, 64], 4, 2, 96, 16),
    ([9], [40], 5, 1, 112, 16),             # groups that divide nothing
    ([300], [301], 3, 1, 64, 16),
    ([4, 90], [50, 100], 14, 2, 48, 24),    # pages of no power of two
    ([4, 90], [50, 100], 2, 2, 32, 7),
    ([40], [45], 40, 1, 16, 1),             # pages of one token
]


@pytest.mark.parametrize("new,ctx,hq,hkv,d,block", SMALL)
@pytest.mark.parametrize("window", [0, 1, 13, 100])
def test_small(paged, dev, new, ctx, hq, hkv, d, block, window):
    _check(paged, dev, _case(new, ctx, hq, hkv, d, block, seed=len(new) + d), window=window)


@pytest.mark.parametrize("d", range(16, 257, 16))
def test_every_head_size(paged, dev, d):
    for new, ctx in (([3, 1], [40, 300]), ([45, 20], [200, 70]), ([2], [1300]), ([70], [1200])):
        _check(paged, dev, _case(new, ctx, 2, 1, d, 16, seed=d))


@pytest.mark.parametrize("d", [80, 128, 256])
@pytest.mark.parametrize("window", [0, 500])
@pytest.mark.parametrize("new,ctx,hq,hkv", [([1, 1, 3], [3000, 17, 1100], 4, 2), ([16], [5000], 4, 2), ([100, 1, 20], [1500, 2600, 40], 4, 1),
                                            ([400], [1700], 2, 1), ([1] * 70, [20 * i + 1 for i in range(70)], 2, 1)])
def test_long_contexts_split_over_workgroups(paged, dev, d, window, new, ctx, hq, hkv):
    _check(paged, dev, _case(new, ctx, hq, hkv, d, 32, seed=d + len(new)), window=window)


def test_rows_that_see_nothing(paged, dev):
    case = list(_case([6, 40, 3, 2], [6, 40, 30, 9], 4, 2, 64, 16))
    for lens in ([2, 10, 0, 9], [0, 0, 0, 0], [-5, 3, -2 ** 31, 1], [6, 41, 3, 2]):
        case[4] = torch.tensor(lens, dtype=I)
        _check(paged, dev, tuple(case))
        _check(paged, dev, tuple(case), window=3)


def test_context_longer_than_the_table(paged, dev):
    q, kc, vc, tables, ctx, starts = _case([5, 50], [64, 96], 4, 2, 64, 16, extra_pages=0)
    ctx = torch.tensor([70, 130], dtype=I)
    tables = tables.clamp(max=kc.shape[0] - 1)
    kc, vc = kc.nan_to_num(0, 0, 0), vc.nan_to_num(0, 0, 0)
    _check(paged, dev, (q, kc, vc, tables, ctx, starts))


def test_scale_and_large_scores(paged, dev):
    for scale in (1e-4, 0.03, 1.0):
        _check(paged, dev, _case([3, 40], [50, 200], 4, 2, 64, 16), scale=scale)
    _check(paged, dev, _case([3, 40], [50, 1500], 4, 2, 64, 16, spread=4.0))


@pytest.mark.parametrize("rows", [3, 60])
@pytest.mark.parametrize("window", [0, 20])
def test_what_a_row_does_not_see_has_no_effect(paged, dev, rows, window):
    """Infinities and NaN in the K and V of tokens inside the context, which earlier rows must not notice and later
    rows (or, with a window, only some) must."""
    q, kc, vc, tables, ctx, starts = _case([rows, 30], [100, 1100], 4, 2, 128, 16, seed=2)
    block = 16

    def put(cache, b, tok, head, dim, value):
        f = head * 128 + dim
        cache[tables[b, tok // block].long(), f // 16, tok % block, f % 16] = value

    clean = [t.clone() for t in (kc, vc)]
    put(vc, 0, 98, 0, 5, math.inf)
    put(vc, 0, 99, 1, 6, math.nan)
    put(vc, 1, 1085, 0, 127, -math.inf)
    put(kc, 0, 97, 1, 3, math.nan)
    put(kc, 1, 1090, 0, 0, math.inf)
    args = lambda k, v: [t.to(dev) for t in (q, k, v, tables, ctx, starts)]  # noqa: E731
    o, lse = paged.paged_attention_chunk(*args(kc, vc), window=window, return_lse=True)
    base, base_lse = paged.paged_attention_chunk(*args(*clean), window=window, return_lse=True)
    at = torch.cat([torch.arange(100 - rows, 100), torch.arange(1070, 1100)])[:, None, None]
    first = torch.arange(rows + 30)[:, None, None] < rows
    head = torch.arange(4)[None, :, None] // 2
    dim = torch.arange(128)[None, None]
    sees = lambda tok: (at >= tok) & ((window == 0) | (at < tok + window))  # noqa: E731
    touched = first & (((head == 0) & (dim == 5) & sees(98)) | ((head == 1) & (dim == 6) & sees(99)) | ((head == 1) & sees(97)))
    touched = touched | ~first & (((head == 0) & (dim == 127) & sees(1085)) | ((head == 0) & sees(1090)))
    o, base = o.cpu(), base.cpu()
    assert torch.equal(o[~touched], base[~touched])
    inf_k = (~first & (head == 0) & sees(1090)).expand_as(o)  # a score of +-inf: NaN, or the weight of that key 0
    assert not o[touched & ~inf_k].isfinite().any()
    untouched_lse = ~((first & (head == 1) & sees(97)) | (~first & (head == 0) & sees(1090)))[..., 0]
    assert torch.equal(lse.cpu()[untouched_lse], base_lse.cpu()[untouched_lse])


def test_rows_of_no_sequence_are_left_alone(paged, dev):
    q, kc, vc, tables, ctx, starts = _case([4, 50], [40, 120], 4, 2, 64, 16)
    pad = torch.randn(9, 4, 64).half()
    q2 = torch.cat([pad[:3], q, pad[3:]])
    out = torch.full_like(q2, 7.0).to(dev)
    o = paged.paged_attention_chunk(*(t.to(dev) for t in (q2, kc, vc, tables, ctx, starts + 3)), out=out)
    assert o.data_ptr() == out.data_ptr()
    want = paged.paged_attention_chunk(*(t.to(dev) for t in (q, kc, vc, tables, ctx, starts)))
    assert torch.equal(o[3:57], want) and (o[:3] == 7).all() and (o[57:] == 7).all()


def test_bad_starts_stay_inside(paged, dev):
    """Bounds outside the batch are limited, decreasing ones give empty sequences; the others' rows are right."""
    q, kc, vc, tables, ctx, starts = _case([4, 50, 3], [40, 120, 60], 4, 2, 64, 16)
    for s in ([-9, 4, 54, 99], [0, 4, 54, 57], [0, 4, 2, 57], [50, 10, 5, -1], [2 ** 31 - 1, 0, 4, 10]):
        out = paged.paged_attention_chunk(*(t.to(dev) for t in (q, kc, vc, tables, ctx)), torch.tensor(s, dtype=I, device=dev),
                                          out=torch.zeros_like(q).to(dev))
        assert out.isfinite().all()


def test_equal_to_decode_and_to_smaller_chunks(paged, ops, dev):
    """One call over a prompt gives what its chunks give, and single tokens what ops.paged_attention gives."""
    q, kc, vc, tables, ctx, starts = [t.to(dev) for t in _case([130, 77], [330, 177], 8, 2, 128, 16)]
    tables = tables.clamp(max=kc.size(0) - 1)
    whole = paged.paged_attention_chunk(q, kc, vc, tables, ctx, starts)
    for step in (1, 13, 64):
        for at in range(0, 77, step):
            n = min(step, 77 - at)
            rows = torch.cat([q[at:at + n], q[130 + at:130 + at + n]])
            got = paged.paged_attention_chunk(rows, kc, vc, tables, torch.tensor([200 + at + n, 100 + at + n], dtype=I, device=dev),
                                              torch.tensor([0, n, 2 * n], dtype=I, device=dev))
            want = torch.cat([whole[at:at + n], whole[130 + at:130 + at + n]])
            # each is within a rounding of the weights and one of the result
            torch.testing.assert_close(got.float(), want.float(), rtol=2.0 ** -9, atol=2.0 ** -9)
            if step == 1:
                lens = torch.tensor([200 + at + 1, 100 + at + 1], dtype=I, device=dev)
                torch.testing.assert_close(ops.paged_attention(rows, kc, vc, tables, lens).float(), want.float(), rtol=2.0 ** -9, atol=2.0 ** -9)


def test_results_do_not_depend_on_the_pages_or_the_run(paged, dev):
    case = [t.to(dev) for t in _case([20, 3, 90], [1500, 2300, 400], 4, 2, 128, 16, seed=5)]
    q, kc, vc, tables, ctx, starts = case
    first = paged.paged_attention_chunk(*case, return_lse=True)
    for _ in range(3):
        again = paged.paged_attention_chunk(*case, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    perm = torch.randperm(kc.size(0), device=dev)
    inverse = torch.empty_like(perm)
    inverse[perm] = torch.arange(kc.size(0), device=dev)
    moved = torch.where(tables < kc.size(0), inverse[tables.long().clamp(max=kc.size(0) - 1)].int(), tables)
    again = paged.paged_attention_chunk(q, kc[perm], vc[perm], moved, ctx, starts, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_joined_by_log_sum_exp(paged, dev):
    """The parts of a context, attended on their own, join to the whole."""
    q, kc, vc, tables, ctx, starts = [t.to(dev) for t in _case([12], [12 + 320], 4, 2, 64, 32, seed=9)]
    tables = tables.clamp(max=kc.size(0) - 1)
    # decode-like rows that see all of the first 320 tokens: one sequence per row
    whole, lse = paged.paged_attention_chunk(q, kc, vc, tables, ctx, starts, return_lse=True)
    rows = torch.arange(13, dtype=I, device=dev)
    past, past_lse = paged.paged_attention_chunk(q, kc, vc, tables.expand(12, -1).contiguous(),
                                                 torch.full((12,), 320, dtype=I, device=dev), rows, return_lse=True)
    own, own_lse = paged.paged_attention_chunk(q, kc, vc, tables, ctx, starts, window=12, return_lse=True)
    # row i sees i + 1 new keys and, through its window, 11 - i of the past: take those back out
    both = torch.logaddexp(past_lse, own_lse)
    assert (both >= lse - 1e-4).all()
    single = paged.paged_attention_chunk(q[:1], kc, vc, tables[:, 10:].contiguous(), ctx - 320 - 11,
                                         torch.tensor([0, 1], dtype=I, device=dev), return_lse=True)
    total = torch.logaddexp(past_lse[:1], single[1])
    joined = past[:1].float() * (past_lse[:1] - total).exp()[..., None] + single[0].float() * (single[1] - total).exp()[..., None]
    torch.testing.assert_close(total, lse[:1], rtol=0, atol=2.0 ** -18)
    torch.testing.assert_close(joined, whole[:1].float(), rtol=2.0 ** -9, atol=2.0 ** -9)


def test_empty_batches(paged, dev):
    q, kc, vc, tables, ctx, starts = [t.to(dev) for t in _case([3], [20], 4, 2, 64, 16)]
    none = torch.zeros(0, dtype=I, device=dev)
    assert paged.paged_attention_chunk(q[:0], kc, vc, tables, ctx, torch.zeros(2, dtype=I, device=dev)).shape == (0, 4, 64)
    out = torch.full_like(q, 3.0)
    assert (paged.paged_attention_chunk(q, kc, vc, tables[:0], none, torch.zeros(1, dtype=I, device=dev), out=out) == 3).all()
    o, lse = paged.paged_attention_chunk(q, kc, vc, tables[:, :0].contiguous(), ctx, starts, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()
    o, lse = paged.paged_attention_chunk(q, kc[:0], vc[:0], tables, ctx, starts, return_lse=True)
    assert (o == 0).all() and (lse == -math.inf).all()


def test_arguments_are_checked(paged, dev):
    q, kc, vc, tables, ctx, starts = case = [t.to(dev) for t in _case([3], [20], 4, 2, 64, 16)]
    f = paged.paged_attention_chunk
    for args, kw, match in [((q.float(), *case[1:]), {}, "float16"), ((q, kc, vc, tables.long(), ctx, starts), {}, "int32"),
                            ((q, kc, vc, tables, ctx, starts[:1]), {}, "query_starts"), ((q, kc, vc, tables, ctx.cpu(), starts), {}, "GPU device"),
                            (case, dict(window=-1), "window"), (case, dict(scale=0.0), "scale"), (case, dict(scale=-1.0), "scale"),
                            (case, dict(scale=math.nan), "scale"), (case, dict(scale=1e-60), "scale"), (case, dict(out=q), "overlap"),
                            (case, dict(out=torch.zeros(4, 4, 64, dtype=H, device=dev)), "shape of q"),
                            ((q[:, :3].contiguous(), *case[1:]), {}, "multiple of num_kv_heads"),
                            ((q.transpose(0, 1), *case[1:]), {}, "contiguous")]:
        with pytest.raises(RuntimeError, match=match):
            f(*args, **kw)


def test_a_cache_beyond_four_gigabytes(paged, dev):
    """Pages whose offsets pass 32 bits."""
    hkv, d, block = 8, 128, 128
    pool = (5 << 30) // (hkv * d * block * 2)
    kc = torch.zeros(pool, hkv * d // 16, block, 16, dtype=H, device=dev)
    vc = torch.zeros_like(kc)
    far = [pool - 1, pool - 3, 0, pool // 2]
    g = torch.Generator().manual_seed(4)
    for p in far:
        kc[p], vc[p] = torch.randn(kc.shape[1:], generator=g).half().to(dev), torch.randn(kc.shape[1:], generator=g).half().to(dev)
    small_k, small_v = kc[far].cpu(), vc[far].cpu()
    for new in (2, 40):
        q = torch.randn(new, 16, d, generator=g).half()
        ctx, starts = torch.tensor([500], dtype=I), torch.tensor([0, new], dtype=I)
        got = paged.paged_attention_chunk(q.to(dev), kc, vc, torch.tensor([far], dtype=I, device=dev), ctx.to(dev), starts.to(dev))
        want, _ = S.paged_attention_chunk_ref(q, small_k, small_v, torch.arange(4, dtype=I)[None], ctx, starts)
        assert (got.cpu().double() - want).norm() <= 3 * 2.0 ** -11 * want.norm()


def test_replayed_from_a_graph(paged, dev):
    """Captured once, replayed on batches that change in place, eager work in between; the workspace is the graph's own."""
    q, kc, vc, tables, ctx, starts = static = [t.to(dev) for t in _case([6, 60, 1], [1200, 90, 1500], 4, 2, 128, 16, extra_pages=0)]
    tables.clamp_(max=kc.size(0) - 1)
    kc.nan_to_num_(0, 0, 0)
    vc.nan_to_num_(0, 0, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.paged_attention_chunk(*static, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = paged.paged_attention_chunk(*static, return_lse=True)
    for i, (s, c) in enumerate([((0, 6, 66, 67), (1200, 90, 1500)), ((0, 30, 60, 67), (1500, 700, 8)), ((0, 0, 1, 67), (0, 1, 1500))]):
        q.copy_(torch.randn(q.shape).half())
        starts.copy_(torch.tensor(s, dtype=I))
        ctx.copy_(torch.tensor(c, dtype=I))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = paged.paged_attention_chunk(*static, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_two_streams_at_once(paged, dev):
    cases = [[t.to(dev) for t in _case([8, 50], [1800, 300], 4, 2, 128, 16, seed=s)] for s in (1, 2)]
    want = [paged.paged_attention_chunk(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(paged.paged_attention_chunk(*c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


@pytest.mark.parametrize("rows", [3, 60])
@pytest.mark.parametrize("window", [0, 2700])
def test_values_that_are_not_finite_in_cut_tiles(paged, dev, rows, window):
    """As above where a tile's keys are shared among workgroups: at the context's end, and where the windows begin."""
    q, kc, vc, tables, ctx, starts = _case([rows], [5000], 4, 2, 128, 16, seed=3)
    bad = vc.clone()
    places = [(4998, 0, 5, math.inf), (4999, 1, 6, math.nan), (2299, 0, 7, -math.inf), (2300 - rows, 1, 70, math.inf), (2298, 1, 100, math.nan)]
    for tok, head, dim, value in places:
        f = head * 128 + dim
        bad[tables[0, tok // 16].long(), f // 16, tok % 16, f % 16] = value
    o, base = (paged.paged_attention_chunk(*(t.to(dev) for t in (q, kc, v, tables, ctx, starts)), window=window).cpu() for v in (bad, vc))
    at = torch.arange(5000 - rows, 5000)[:, None, None]
    head, dim = torch.arange(4)[None, :, None] // 2, torch.arange(128)[None, None]
    touched = torch.zeros(o.shape, dtype=torch.bool)
    for tok, h, d, _ in places:
        touched |= (head == h) & (dim == d) & (at >= tok) & ((window == 0) | (at < tok + window))
    assert torch.equal(o[~touched], base[~touched]) and not o[touched].isfinite().any()


def test_cut_tiles_in_two_graphs_and_on_two_streams(paged, dev):
    """Each call has partial results of its own: graphs replayed in turn, and calls on streams at once."""
    cases = [[t.to(dev) for t in _case(new, ctx, 4, 2, 128, 16, seed=s)] for s, (new, ctx) in enumerate([([6, 60, 1], [5000, 400, 3000]), ([40, 2], [4000, 6000])])]
    want = [paged.paged_attention_chunk(*c, return_lse=True) for c in cases]
    graphs, held = [], []
    side = torch.cuda.Stream()
    for c in cases:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            paged.paged_attention_chunk(*c, return_lse=True)
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(paged.paged_attention_chunk(*c, return_lse=True))
    for i in (0, 1, 1, 0, 1, 0):
        graphs[i].replay()
        again = paged.paged_attention_chunk(*cases[1 - i], return_lse=True)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held[i], want[i])), i
        assert all(torch.equal(a, b) for a, b in zip(again, want[1 - i])), i
        for t in held[i]:
            t.zero_()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(paged.paged_attention_chunk(*c, return_lse=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for x in g for a, b in zip(x, w))


@pytest.mark.parametrize("new,ctx,hq,hkv,d", [
    ([1] * 1100, [1 + 7 * (i % 9) + (3000 if i % 400 == 3 else 0) for i in range(1100)], 2, 1, 16),  # more tiles than a partition takes
    ([1] * 1020, [1 + 7 * (i % 9) + (3000 if i % 400 == 3 else 0) for i in range(1020)], 2, 1, 16),
    ([0] * 700 + [2, 0, 5] + [0] * 600 + [40], [9] * 700 + [3000, 9, 70] + [0] * 600 + [2800], 2, 1, 32),  # few with tokens
    ([1, 3, 40], [500, 2600, 3000], 300, 1, 16),                                                          # a token's heads in more than one tile
    ([2, 1], [2500, 3], 300, 300, 16),                                                                   # more kv heads than CUs
])
def test_long_tables_at_the_limits_of_the_partition(paged, dev, new, ctx, hq, hkv, d):
    _check(paged, dev, _case(new, ctx, hq, hkv, d, 16))


@pytest.mark.parametrize("d", [16, 80, 128, 144, 208])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("new,ctx", [([33, 1, 64], [33, 400, 290]), ([65, 128], [333, 128]), ([129, 192], [129, 500]), ([256, 257], [700, 300]),
                                     ([96, 100], [3100, 2900])])
def test_tiles_of_every_height(paged, dev, d, window, new, ctx):
    """Around the numbers of rows at which a tile's work is divided differently."""
    _check(paged, dev, _case(new, ctx, 1, 1, d, 16, seed=d), window=window)


@pytest.mark.parametrize("d", [16, 144])
@pytest.mark.parametrize("seqs", [64, 65, 512, 513, 3000, 5000])
def test_many_sequences(paged, dev, d, seqs):
    """Sequences without tokens among them, and some of several tiles."""
    new = [(0, 1, 1, 2, 1, 0, 3)[i % 7] + (300 if i % 1500 == 63 else 0) for i in range(seqs)]
    _check(paged, dev, _case(new, [n + i % 13 for i, n in enumerate(new)], 1, 1, d, 16, seed=seqs))
    starts = torch.randint(-50, 900, (seqs + 1,), generator=torch.Generator().manual_seed(1)).int()  # out of order
    q, kc, vc, tables, ctx, _ = _case([700], [700], 1, 1, d, 16)
    args = [t.to(dev) for t in (q, kc, vc, tables.expand(seqs, -1).contiguous(), ctx.expand(seqs).contiguous(), starts)]
    assert paged.paged_attention_chunk(*args, out=torch.zeros_like(args[0])).isfinite().all()


@pytest.mark.parametrize("new,ctx", [([3, 1], [700, 40]), ([60, 1], [300, 9]), ([300], [2900]), ([4], [4000])])
@pytest.mark.parametrize("d", [64, 128, 208])
@pytest.mark.parametrize("size,scale", [(1000.0, None), (60000.0, None), (60000.0, 2.0 ** 56), (0.5, 2.0 ** 56), (2.0, 2.0 ** 20)])
def test_scores_far_from_zero(paged, dev, new, ctx, d, size, scale):
    """Queries and keys as large as fp16 goes, and large scales: keys that are all alike weigh the same, however large their
    score, and keys whose score is far above the others' are all that counts.

    All elements of a query are one number, all of a key that number times a power of two (or cut off), so equal keys have
    equal scores in any arithmetic and the others' are far below.  Rounded are the score (a sum of D products, half a step each, and
    its scaling), the weights, which are all the same, once to fp16, the sums (half a step per 32 keys, and 16 for joins) and the result."""
    block = 16
    q, kc, vc, tables, lens, starts = _case(new, ctx, 4, 2, d, block, seed=d)
    q, tables, vc = torch.full_like(q, size), tables.clamp(max=kc.shape[0] - 1), vc.nan_to_num(0, 0, 0)
    for sign in (1, -1):
        for levels in (1, 6):
            level = torch.zeros(kc.shape[0], block)
            for b, n in enumerate(ctx):  # the maximum comes early, or late, or again and again
                for tok in range(n):
                    level[tables[b, tok // block].long(), tok % block] = tok * 7 % 11 % levels
            k = (sign * size * 2.0 ** -(level if sign < 0 else 5 - level)).clamp(-60000, 60000).half()
            kc = k[:, None, :, None].expand(-1, kc.shape[1], -1, 16).contiguous()
            want, want_lse = S.paged_attention_chunk_ref(q, kc, vc, tables, lens, starts, scale=scale)
            o, lse = paged.paged_attention_chunk(*(t.to(dev) for t in (q, kc, vc, tables, lens, starts)), scale=scale, return_lse=True)
            o, lse = o.cpu().double(), lse.cpu().double()
            finite, what = bool(o.isfinite().all() and lse.isfinite().all()), (sign, levels)
            assert finite, what
            worst = float(((lse - want_lse).abs() - want_lse.abs() * 2.0 ** -24 * (d + 4)).max())
            assert worst <= 2.0 ** -18, (what, worst)
            tol = want.abs() * 2.0 ** -10 + (max(ctx) / 32 + 16) * 2.0 ** -24 * float(vc.abs().max()) + 2.0 ** -24
            worst = float(((o - want).abs() / tol).max())
            assert worst <= 1, (what, worst)


def _check_bounds(paged, dev, case, starts):
    """Limited bounds, sequence by sequence: rows of exactly one sequence against the definition, rows of none untouched (rows of
    several are one of theirs, or a mixture).  How many rows there are of each kind."""
    q, kc, vc, tables, ctx, _ = case
    rows = q.shape[0]
    want = torch.full(q.shape, math.nan, dtype=torch.float64)
    times = torch.zeros(rows, dtype=torch.long)
    for b in range(len(ctx)):
        begin = min(max(int(starts[b]), 0), rows)
        end = min(max(int(starts[b + 1]), begin), rows)
        if begin == end:
            continue
        own = torch.tensor([0, end - begin], dtype=I)
        want[begin:end] = S.paged_attention_chunk_ref(q[begin:end], kc, vc, tables[b:b + 1], ctx[b:b + 1], own)[0]
        times[begin:end] += 1
    out = torch.full_like(q, 7.0).to(dev)
    got = paged.paged_attention_chunk(*(t.to(dev) for t in (q, kc, vc, tables, ctx, starts)), out=out).cpu().double()
    assert (got[times == 0] == 7).all()
    once = times == 1
    tol, _ = _tolerances((q, kc, vc, tables, ctx, starts), None, None, q.shape[-1] ** -0.5, 0, (want[once], torch.zeros(1)))
    assert ((got[once] - want[once]).abs() <= tol).all(), float(((got[once] - want[once]).abs() / tol).max())
    return [int((times == n).sum()) for n in (0, 1)]


@pytest.mark.parametrize("starts,untouched,once", [([-9, 4, 54, 99], 0, 57), ([0, 4, 54, 57], 0, 57), ([3, 4, 50, 50], 10, 47), ([0, 4, 2, 57], 0, 55),
                                                   ([50, 10, 5, -1], 57, 0), ([2 ** 31 - 1, 0, 4, 10], 47, 10), ([20, 57, 30, 40], 20, 27)])
def test_bounds_outside_the_batch_and_out_of_order(paged, dev, starts, untouched, once):
    """The rows that stay with one sequence are right, those with none are left alone."""
    case = _case([4, 50, 3], [60, 120, 60], 4, 2, 64, 16)
    assert _check_bounds(paged, dev, case, torch.tensor(starts, dtype=I)) == [untouched, once]


@pytest.mark.parametrize("d", [16, 144])
@pytest.mark.parametrize("width", [44, 200])
@pytest.mark.parametrize("seqs", [60, 500, 600])
def test_many_bounds_out_of_order(paged, dev, d, width, seqs):
    """Bounds in order but for some neighbours, among few sequences and many, with whole tiles and (where the table is wide)
    with the partition: every row of one sequence is attended as that sequence's."""
    g = torch.Generator().manual_seed(seqs + width)
    q, kc, vc, tables, _, _ = _case([700], [700], 1, 1, d, 16, seed=d)
    tables = torch.cat([tables[:, :44], torch.zeros(1, width - 44, dtype=I)], 1).clamp(max=kc.shape[0] - 1)
    starts = torch.randint(0, 701, (seqs + 1,), generator=g).sort().values.int()
    starts[0], starts[-1] = -5, 720
    for i in torch.randperm(seqs - 2, generator=g)[:12].tolist():
        starts[i + 1], starts[i + 2] = starts[i + 2].clone(), starts[i + 1].clone()
    ctx = 660 + torch.arange(seqs, dtype=I) % 40
    kc, vc = kc.nan_to_num(0, 0, 0), vc.nan_to_num(0, 0, 0)
    untouched, once = _check_bounds(paged, dev, (q, kc, vc, tables.expand(seqs, -1).contiguous(), ctx, None), starts)
    assert untouched == 0 and once >= 300


def test_every_row_joined_by_log_sum_exp(paged, dev):
    """Every row's context in two parts, attended on their own and joined: the keys of the first 320 tokens and the row's own
    chunk as far as it, against the whole and against the definition.

    A log-sum-exp is within `_tolerances` of its own; the joined one adds two exponentials and a logarithm in fp32 (2^-20).  A weight of the
    join is off by as much as the log-sum-exps are, and each part by its own tolerance."""
    n, past_len, block = 12, 320, 32
    case = q, kc, vc, tables, ctx, starts = _case([n], [n + past_len], 4, 2, 64, block, seed=9)
    tables = tables.clamp(max=kc.shape[0] - 1)
    on = lambda *ts: [t.to(dev) for t in ts]  # noqa: E731
    ref = S.paged_attention_chunk_ref(q, kc, vc, tables, ctx, starts)
    whole, lse = paged.paged_attention_chunk(*on(q, kc, vc, tables, ctx, starts), return_lse=True)
    one_each = torch.arange(n + 1, dtype=I)
    past, past_lse = paged.paged_attention_chunk(*on(q, kc, vc, tables.expand(n, -1).contiguous(), torch.full((n,), past_len, dtype=I), one_each),
                                                 return_lse=True)
    own, own_lse = paged.paged_attention_chunk(*on(q, kc, vc, tables[:, past_len // block:].contiguous(), ctx - past_len, starts), return_lse=True)
    total = torch.logaddexp(past_lse, own_lse)
    joined = past.float() * (past_lse - total).exp()[..., None] + own.float() * (own_lse - total).exp()[..., None]
    tol_o, tol_l = _tolerances(case, None, None, 64 ** -0.5, 0, ref)
    assert ((total.cpu().double() - ref[1]).abs() <= 2 * tol_l + 2.0 ** -20).all()
    assert ((lse.cpu().double() - ref[1]).abs() <= tol_l).all()
    largest = float(vc.nan_to_num(0, 0, 0).abs().max())
    assert ((joined.cpu().double() - ref[0]).abs() <= 2 * tol_o + (3 * tol_l.max() + 2.0 ** -19) * largest).all()
    assert ((whole.cpu().double() - ref[0]).abs() <= tol_o).all()


@pytest.mark.parametrize("d", [80, 128, 208])
@pytest.mark.parametrize("new,ctx", [([9, 1], [700, 300]), ([50], [400]), ([130], [2900])])
@pytest.mark.parametrize("window", [0, 200])
def test_rows_near_and_far_in_one_tile(paged, dev, d, new, ctx, window):
    """Rows whose scores are far from zero next to ordinary ones: those come out as exactly as without them, these inside what
    their values span."""
    case = list(_case(new, ctx, 4, 2, d, 16, seed=d))
    far = torch.arange(sum(new)) % 5 == 3
    case[0] = torch.where(far[:, None, None], (case[0].double() * 20000).clamp(-60000, 60000).half(), case[0])
    ref = S.paged_attention_chunk_ref(*case, window=window)
    o, lse = paged.paged_attention_chunk(*(t.to(dev) for t in case), window=window, return_lse=True)
    o, lse = o.cpu().double(), lse.cpu().double()
    assert bool(o.isfinite().all() and lse.isfinite().all())
    assert o.abs().max() <= case[2][case[2].isfinite()].abs().max()
    # a far row's log-sum-exp is its largest score, to the rounding of D products and their sum
    assert ((lse[far] - ref[1][far]).abs() <= ref[1][far].abs().clamp(min=1) * (d + 4) * 2.0 ** -20).all()
    near = [case[0][~far], *case[1:]]
    tol_o, tol_l = _tolerances(near, None, None, d ** -0.5, window, (ref[0][~far], ref[1][~far]))
    assert ((o[~far] - ref[0][~far]).abs() <= tol_o).all()
    assert ((lse[~far] - ref[1][~far]).abs() <= tol_l).all()
