"""Pages of the paged caches, copied, forked, given out, freed and packed on the device, against the same steps on Python
lists.  Everything is exact."""
import random

import pytest
import torch

import oracle.serving_ref as S

pytestmark = pytest.mark.gpu
H, I = torch.float16, torch.int32


@pytest.fixture(scope="module")
def paged():
    from ascend910a_extras import paged as p

    return p


def _caches(dev, blocks, row, block, layers, seed=0):
    g = torch.Generator().manual_seed(seed)
    # bit patterns of every kind, NaN among them: pages are moved, not computed with
    return [torch.randint(-32768, 32768, (blocks, row // 16, block, 16), generator=g, dtype=torch.int16).view(H).to(dev)
            for _ in range(2 * layers)]


def _same_bits(a, b):
    return torch.equal(a.cpu().view(torch.int16), b.cpu().view(torch.int16))


def _pool(seed, blocks, block, seqs, width, share=0.3, odd=True):
    """Tables, lengths and counts of a pool in use: shared pages, rows of length zero, lengths beyond the row, entries and
    counts that are out of range."""
    r = random.Random(seed)
    tables = [[r.randrange(-2, blocks + 2) if odd else -1 for _ in range(width)] for _ in range(seqs)]
    order = list(range(blocks))
    r.shuffle(order)
    counts = [0] * blocks
    lens = []
    for b in range(seqs):
        n = r.choice([0, 1, block, block + 1, r.randrange(0, width * block + 1), r.randrange(0, width * block + 1)])
        for j in range(-(-n // block)):
            if b and r.random() < share:
                page = tables[r.randrange(b)][j]
            elif order:
                page = order.pop()
            else:
                n = min(n, j * block)
                break
            tables[b][j] = page
            if 0 <= page < blocks:
                counts[page] += 1
        lens.append(n)
    if odd:
        lens[r.randrange(seqs)] = r.choice([-3, width * block + 5])
        counts = [c if c else r.choice([0, 0, -1, -7]) for c in counts]
    return tables, lens, counts


def _dev(dev, *lists):
    return [torch.tensor(x, dtype=I, device=dev) for x in lists]


POOLS = [(1, 16, 1, 1), (7, 16, 3, 3), (64, 16, 9, 12), (300, 32, 40, 9), (4096, 16, 60, 50), (4097, 16, 60, 50), (8192, 8, 200, 33), (8193, 16, 33, 40), (20000, 1, 65, 200)]


@pytest.mark.parametrize("row,block,blocks,layers,pairs", [(64, 16, 9, 1, 3), (48, 7, 33, 2, 16), (1024, 128, 24, 3, 11), (16, 1, 5, 1, 2)])
def test_copy(paged, dev, row, block, blocks, layers, pairs):
    caches = _caches(dev, blocks, row, block, layers)
    order = torch.randperm(blocks)[: 2 * pairs].tolist()
    src, dst = order[:pairs] + [-1, blocks, 0, 1], order[pairs:2 * pairs] + [0, 1, blocks, -5]
    want = [c.clone() for c in caches]
    for s, d in zip(src, dst):
        if 0 <= s < blocks and 0 <= d < blocks:
            for w, c in zip(want, caches):
                w[d] = c[s]
    s, d = _dev(dev, src, dst)
    assert paged.copy_pages(caches[:layers], caches[layers:], s, d) is None
    assert all(_same_bits(a, b) for a, b in zip(caches, want))
    paged.copy_pages(caches[:layers], caches[layers:], s[:0], d[:0])
    paged.copy_pages(caches[:layers], [], s[-4:], d[-4:])
    assert all(_same_bits(a, b) for a, b in zip(caches, want))


@pytest.mark.parametrize("blocks,block,seqs,width", POOLS)
@pytest.mark.parametrize("children", [1, 5, 70])
def test_fork(paged, dev, blocks, block, seqs, width, children):
    for seed in range(3):
        tables, lens, counts = _pool(seed, blocks, block, seqs, width)
        r = random.Random(seed + 99)
        parents = [r.randrange(-1, seqs + 1) for _ in range(children)]
        if seed == 2:  # a pool that is nearly full
            counts = [c if r.random() < 4 / blocks or c > 0 else 1 for c in counts]
        caches = _caches(dev, blocks, 32, block, 2, seed)
        ref = S.PoolRef(counts, block)
        rows, out_lens = ref.fork(tables, lens, parents)
        t, l, p, c = _dev(dev, tables, lens, parents, counts)
        keep = [x.clone() for x in (t, l, p, c)]
        want = [ref.moved(x.cpu()) for x in caches]
        got = paged.fork_sequences(t, l, p, c, caches[:2], caches[2:])
        assert got[0].tolist() == rows and got[1].tolist() == out_lens and got[2].tolist() == ref.counts
        assert all(_same_bits(a, b) for a, b in zip(caches, want))
        assert all(torch.equal(a, b) for a, b in zip(keep, (t, l, p, c)))


@pytest.mark.parametrize("blocks,block,seqs,width", POOLS)
def test_extend(paged, dev, blocks, block, seqs, width):
    for seed in range(4):
        tables, lens, counts = _pool(seed + 10, blocks, block, seqs, width)
        r = random.Random(seed + 5)
        wanted = [r.choice([n + 1, n, 0, -1, width * block, width * block + 1, 2 ** 31 - 1, n + r.randrange(3 * block)]) for n in lens]
        ref = S.PoolRef(counts, block)
        rows, granted = ref.extend(tables, lens, wanted)
        t, l, w, c = _dev(dev, tables, lens, wanted, counts)
        got = paged.extend_sequences(t, l, w, c, block)
        assert got[0].tolist() == rows and got[1].tolist() == granted and got[2].tolist() == ref.counts
        assert t.tolist() == tables and c.tolist() == counts


@pytest.mark.parametrize("blocks,block,seqs,width", POOLS)
def test_free(paged, dev, blocks, block, seqs, width):
    for seed in range(3):
        tables, lens, counts = _pool(seed + 20, blocks, block, seqs, width)
        r = random.Random(seed)
        which = [r.randrange(-2, seqs + 2) for _ in range(r.choice([0, 1, seqs, 3 * seqs]))]  # the same one several times too
        ref = S.PoolRef(counts, block)
        ref.free(tables, lens, which)
        t, l, w, c = _dev(dev, tables, lens, which, counts)
        assert paged.free_sequences(t, l, w, c, block).tolist() == ref.counts
        assert c.tolist() == counts


@pytest.mark.parametrize("blocks,block,seqs,width", POOLS)
def test_compact(paged, dev, blocks, block, seqs, width):
    for seed in range(3):
        tables, lens, counts = _pool(seed + 30, blocks, block, seqs, width)
        if seed == 1:
            counts = [max(c, 1) for c in counts]  # nothing free
        if seed == 2:
            counts = [0] * blocks                 # nothing used
        ref = S.PoolRef(counts, block)
        rows, used = ref.compact(tables, lens)
        caches = _caches(dev, blocks, 48, block, 1, seed)
        want = [ref.moved(x.cpu()) for x in caches]
        t, l, c = _dev(dev, tables, lens, counts)
        got = paged.compact_pages(t, l, c, caches[:1], caches[1:])
        assert got[0].tolist() == rows and got[1].tolist() == ref.counts and got[2].tolist() == [used]
        assert all(_same_bits(a, b) for a, b in zip(caches, want))
        assert t.tolist() == tables and c.tolist() == counts


def test_many_layers_and_pages_larger_than_a_copy_step(paged, dev):
    blocks, block, row = 12, 160, 1024
    caches = _caches(dev, blocks, row, block, 3)
    tables, lens, counts = [[4, 9], [7, 2]], [159, 201], [0] * blocks
    for row_, n in zip(tables, lens):
        for j in range(-(-n // block)):
            counts[row_[j]] = 1
    ref = S.PoolRef(counts, block)
    rows, out = ref.fork(tables, lens, [1, 0, 1])
    want = [ref.moved(x.cpu()) for x in caches]
    t, l, p, c = _dev(dev, tables, lens, [1, 0, 1], counts)
    got = paged.fork_sequences(t, l, p, c, caches[:3], caches[3:])
    assert got[0].tolist() == rows and got[1].tolist() == out
    assert all(_same_bits(a, b) for a, b in zip(caches, want))


@pytest.mark.parametrize("requests", [255, 256, 257, 300, 600, 1100])
@pytest.mark.parametrize("blocks", [700, 4096])
def test_more_requests_than_threads(paged, dev, requests, blocks):
    """One launch up to 256 requests, two beyond; pools that run dry in the middle of the requests."""
    block, width = 4, 27
    tables, lens, counts = _pool(requests, blocks, block, 50, width, odd=False)
    r = random.Random(requests)
    parents = [r.randrange(50) for _ in range(requests)]
    ref = S.PoolRef(counts, block)
    rows, out = ref.fork(tables, lens, parents)
    caches = _caches(dev, blocks, 16, block, 1)
    want = [ref.moved(x.cpu()) for x in caches]
    t, l, p, c = _dev(dev, tables, lens, parents, counts)
    got = paged.fork_sequences(t, l, p, c, caches[:1], caches[1:])
    assert got[0].tolist() == rows and got[1].tolist() == out and got[2].tolist() == ref.counts
    assert all(_same_bits(a, b) for a, b in zip(caches, want))
    wanted = [n + r.choice([0, 1, 5, 40]) for n in out]
    room, granted = ref.extend(rows, out, wanted)
    more = paged.extend_sequences(got[0], got[1], _dev(dev, wanted)[0], got[2], block)
    assert more[0].tolist() == room and more[1].tolist() == granted and more[2].tolist() == ref.counts
    ref.free(room, granted, range(requests))
    assert paged.free_sequences(more[0], more[1], _dev(dev, list(range(requests)))[0], more[2], block).tolist() == ref.counts


@pytest.mark.parametrize("blocks", [60, 4200])
def test_a_beam_step_in_a_graph(paged, dev, blocks):
    """Fork, extend, free and pack captured once, on one stream, and replayed on pools that change in place."""
    block, seqs, width = 16, 5, 8
    state = _dev(dev, *_pool(0, blocks, block, seqs, width, odd=False))
    parents, rows_all = _dev(dev, [0, 0, 3, 1], list(range(seqs)))
    caches = _caches(dev, blocks, 32, block, 1)
    start = [x.clone() for x in caches]
    wanted = torch.zeros(4, dtype=I, device=dev)

    def step():
        rows, lens, counts = paged.fork_sequences(*state[:2], parents, state[2], caches[:1], caches[1:])
        room, granted, counts = paged.extend_sequences(rows, lens, wanted, counts, block)
        counts = paged.free_sequences(*state[:2], rows_all, counts, block)
        return [rows, lens, room, granted, *paged.compact_pages(room, granted, counts, caches[:1], caches[1:])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(5):
        tables, lens, counts = _pool(seed, blocks, block, seqs, width, odd=False)
        for s, v in zip(state, (tables, lens, counts)):
            s.copy_(torch.tensor(v, dtype=I))
        wanted.copy_(torch.tensor([lens[p] + 1 for p in (0, 0, 3, 1)], dtype=I))
        for x, y in zip(caches, start):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        after = [x.clone() for x in caches]
        for x, y in zip(caches, start):
            x.copy_(y)
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
        assert all(_same_bits(a, b) for a, b in zip(after, caches))
        ref = S.PoolRef(counts, block)
        rows, out = ref.fork(tables, lens, [0, 0, 3, 1])
        room, granted = ref.extend(rows, out, wanted.tolist())
        ref.free(tables, lens, range(seqs))
        first, ref.moves = ref.moved(start[0].cpu()), []
        packed, used = ref.compact(room, granted)
        assert [x.tolist() for x in got] == [rows, out, room, granted, packed, ref.counts, [used]]
        assert _same_bits(after[0], ref.moved(first))


@pytest.mark.parametrize("blocks", [60, 4200])
def test_two_streams_at_once(paged, dev, blocks):
    """Two pools' calls side by side."""
    pools = [_dev(dev, *_pool(s, blocks, 16, 5, 8, odd=False)) for s in (0, 1)]
    caches = [_caches(dev, blocks, 32, 16, 1, seed=s) for s in (0, 1)]
    parents, wanted = _dev(dev, [0, 0, 3, 1], [100] * 5)

    def step(i):
        t, l, c = pools[i]
        rows, lens, counts = paged.fork_sequences(t, l, parents, c, caches[i][:1], caches[i][1:])
        counts = paged.free_sequences(rows, lens, parents, counts, 16)
        return [rows, lens, counts, *paged.extend_sequences(t, l, wanted, c, 16)]

    want = [step(i) for i in (0, 1)]
    streams, got = [torch.cuda.Stream() for _ in pools], [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for x in g for a, b in zip(x, w))


@pytest.mark.parametrize("blocks,children,pages", [(4096, 1, 4000), (4096, 1, 1000), (4096, 4, 1000), (4096, 16, 250), (4000, 7, 580), (4096, 256, 11),
                                                   (4096, 4, 4000), (4096, 16, 1000), (4096, 256, 60)])
def test_children_of_long_parents_in_a_small_pool(paged, dev, blocks, children, pages):
    """Shared pages are counted by (child, page): children of one parent and of several, refused ones and parents that
    are none among them, more pairs than a workgroup looks at in one round."""
    block, seqs = 16, max(1, min(3, blocks // pages))
    width = pages + 5
    r = random.Random(pages + children)
    order = r.sample(range(blocks), pages * seqs)
    tables = [order[b * pages:(b + 1) * pages] + [-1] * (width - pages) for b in range(seqs)]
    lens = [pages * block - (0, 5, block - 1)[b] for b in range(seqs)]
    counts = [0] * blocks
    for p in order:
        counts[p] += 1
    for free in (2, blocks):  # all but two of the free pages are given away first: some children get none
        kept = 0
        for p in range(blocks):
            if counts[p] == 0:
                kept += 1
                counts[p] = 0 if kept <= free else 1
        parents = [r.randrange(-1, seqs + 1) if children > 1 else seqs - 1 for _ in range(children)]
        ref = S.PoolRef(counts, block)
        rows, out = ref.fork(tables, lens, parents)
        caches = _caches(dev, blocks, 16, block, 1)
        want = [ref.moved(x.cpu()) for x in caches]
        t, l, p, c = _dev(dev, tables, lens, parents, counts)
        got = paged.fork_sequences(t, l, p, c, caches[:1], caches[1:])
        assert got[0].tolist() == rows and got[1].tolist() == out and got[2].tolist() == ref.counts
        assert all(_same_bits(a, b) for a, b in zip(caches, want))


def _microseconds(f, calls=20, rounds=7):
    """Median over rounds of the time of a call among others."""
    f()
    times = []
    for _ in range(rounds):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        for _ in range(calls):
            f()
        end.record()
        end.synchronize()
        times.append(begin.elapsed_time(end) * 1000 / calls)
    return sorted(times)[rounds // 2]


@pytest.mark.parametrize("op", ["fork", "free"])
@pytest.mark.parametrize("rows,pages", [(1, 4000), (4, 1000), (16, 1000)])
def test_one_launch_is_not_far_slower_than_two(paged, dev, op, rows, pages):
    """Long sequences cost about the same on both sides of the largest pool that takes one launch (a fork 25 times as
    much where one thread walked all pages of a child)."""
    us = []
    for blocks in (4096, 4097):
        caches = _caches(dev, blocks, 16, 16, 1)
        tables = [[j for j in range(pages)] + [-1] * 8]
        counts = [1] * pages + [0] * (blocks - pages)
        t, l, p, c = _dev(dev, tables, [pages * 16 - 5], [0] * rows, counts)
        if op == "fork":
            us.append(_microseconds(lambda: paged.fork_sequences(t, l, p, c, caches[:1], caches[1:])))
        else:
            us.append(_microseconds(lambda: paged.free_sequences(t, l, p, c, 16)))
    assert us[0] < 4 * us[1], us


@pytest.mark.parametrize("blocks", [60, 5000])
def test_lengths_outside_their_rows_come_back_limited(paged, dev, blocks):
    """A present length counts as far as the row can hold it, from 0 on; whatever is wanted, the row is full or empty."""
    block, width = 16, 4
    t, l, w, c = _dev(dev, [[0, 1, 2, 3], [4, 5, 6, 7], [-1] * 4, [-1] * 4, [8, 9, -1, -1]], [64 + 9, 2 ** 31 - 1, -3, -2 ** 31, 20],
                      [80, 10, 17, 0, 5], [1] * 10 + [0] * (blocks - 10))
    tables, lens, counts = paged.extend_sequences(t, l, w, c, block)
    assert lens.tolist() == [64, 64, 17, 0, 20]
    assert tables.tolist() == [[0, 1, 2, 3], [4, 5, 6, 7], [10, 11, -1, -1], [-1] * 4, [8, 9, -1, -1]]
    assert counts.tolist() == [1] * 12 + [0] * (blocks - 12)


def test_pages_beyond_four_gigabytes(paged, dev):
    """Offsets that pass 32 bits, in bytes and in elements: copies, a fork and packing at the far end of a cache of 9 GiB."""
    row, block = 1024, 128
    blocks = (9 << 30) // (row * block * 2)  # 36864 pages of 256 KiB
    kc = torch.zeros(blocks, row // 16, block, 16, dtype=H, device=dev)
    vc = torch.zeros_like(kc)
    g = torch.Generator().manual_seed(8)

    def fill(*pages):
        for p in pages:
            for c in (kc, vc):
                c[p] = torch.randint(-32768, 32768, c.shape[1:], generator=g, dtype=torch.int16).view(H).to(dev)

    far, middle = blocks - 1, blocks - 2 - (4 << 30) // (row * block * 2)
    fill(far, 3)
    s, d = _dev(dev, [far, 3], [middle, far - 1])
    paged.copy_pages([kc], [vc], s, d)
    for c in (kc, vc):
        assert _same_bits(c[middle], c[far]) and _same_bits(c[far - 1], c[3]) and not c[far - 2].any() and not c[0].any()
    # a child of a parent whose last page is the far one, into the only free pages, both far out too
    counts = torch.ones(blocks, dtype=I, device=dev)
    counts[far - 1] = counts[far - 2] = 0
    kc[far - 1], vc[far - 1] = 0, 0
    t, l, p = _dev(dev, [[middle, far]], [block + 77], [0, 0])
    rows, lens, after = paged.fork_sequences(t, l, p, counts, [kc], [vc])
    assert rows.tolist() == [[middle, far - 2], [middle, far - 1]] and lens.tolist() == [block + 77] * 2
    assert after[middle] == 3 and after[far - 1] == after[far - 2] == 1
    for c in (kc, vc):
        for page in (far - 2, far - 1):
            assert _same_bits(c[page, :, :77], c[far, :, :77]) and not c[page, :, 77:].any()
    # the far pages to the lowest ones
    counts.zero_()
    counts[far], counts[middle], counts[1] = 1, 2, 1
    want = [(c[middle].clone(), c[far].clone()) for c in (kc, vc)]
    kept = kc[1].clone()
    rows, after, used = paged.compact_pages(*_dev(dev, [[middle, far], [1, middle]], [block + 77, block + 1]), counts, [kc], [vc])
    assert rows.tolist() == [[0, 2], [1, 0]] and used.item() == 3 and after[:4].tolist() == [2, 1, 1, 0] and not after[4:].any()
    for c, (first, second) in zip((kc, vc), want):
        assert _same_bits(c[0], first) and _same_bits(c[2], second)
    assert _same_bits(kc[1], kept)
