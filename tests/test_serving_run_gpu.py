"""A server's run over the paged caches with the operators together: prompts and drafted tokens in chunks, beams forked,
decoding, sequences released, the pool packed; a fused projection is rotated in place of its heads, two layers share the
tables.  Attention is compared with its definition in 64 bits over a history kept on the host, the pages with a host that
follows without asking."""
import math

import pytest
import torch

import oracle.serving_ref as S

pytestmark = pytest.mark.gpu
H, I = torch.float16, torch.int32
HQ, HK, D, BLOCK, LAYERS, PAGES, WIDTH, ROTARY = 8, 2, 128, 16, 2, 96, 20, 64


def _attend(q, k, v):
    """The last q.shape[0] tokens of a history k, v; fp64."""
    n, length = q.shape[0], k.shape[0]
    k, v = (x.double().repeat_interleave(HQ // HK, dim=1) for x in (k, v))
    s = torch.einsum("ihd,jhd->hij", q.double(), k) / math.sqrt(D)
    hidden = torch.arange(length)[None, :] > torch.arange(length - n, length)[:, None]
    return torch.einsum("hij,jhd->ihd", s.masked_fill(hidden, -math.inf).softmax(-1), v)


def _tolerance(want, q, k, v):
    """A score's products and sums (D + 4 half steps of its largest size), each weight's rounding to fp16 and its
    exponential (2^-11 and 2^-21), sums in fp32 (half a step per 32 keys), the result's rounding."""
    size = min(float(q.abs().max()) * float(k.abs().max()) * math.sqrt(D), 60.0)
    weight = 2.0 ** -11 + 2.0 ** -21 + 3 * size * (D + 4) * 2.0 ** -24 + (k.shape[0] / 32 + 8) * 2.0 ** -23
    return want.abs() * (2.0 ** -11 + weight) + weight * float(v.abs().max()) + 2.0 ** -24


class Server:
    def __init__(self, dev):
        from ascend910a_extras import ops, paged, rotary

        self.ops, self.paged, self.rotary, self.dev = ops, paged, rotary, dev
        self.caches = [[torch.full((PAGES, HK * D // 16, BLOCK, 16), math.nan, dtype=H, device=dev) for _ in range(LAYERS)]
                       for _ in range(2)]
        self.counts = torch.zeros(PAGES, dtype=I, device=dev)
        self.cos, self.sin = rotary.rotary_tables(WIDTH * BLOCK, ROTARY, scaling="yarn", factor=4.0,
                                                  original_max_position=80, dtype=torch.float32, device=dev)
        self.gen = torch.Generator().manual_seed(11)
        self.tables = torch.full((0, WIDTH), -1, dtype=I, device=dev)
        self.lens = torch.zeros(0, dtype=I, device=dev)
        self.history = []  # per sequence and layer: k, v
        self.pool, self.host_tables, self.host_lens = S.PoolRef([0] * PAGES, BLOCK), [], []

    def _same_pool(self):
        assert self.tables.tolist() == self.host_tables and self.lens.tolist() == self.host_lens
        assert self.counts.tolist() == self.pool.counts

    def add(self, n):
        self.tables = torch.cat([self.tables, torch.full((n, WIDTH), -1, dtype=I, device=self.dev)])
        self.lens = torch.cat([self.lens, torch.zeros(n, dtype=I, device=self.dev)])
        self.history += [[(torch.zeros(0, HK, D, dtype=H),) * 2 for _ in range(LAYERS)] for _ in range(n)]
        self.host_tables, self.host_lens = self.host_tables + [[-1] * WIDTH for _ in range(n)], self.host_lens + [0] * n

    def fork(self, parents):
        t, l, self.counts = self.paged.fork_sequences(self.tables, self.lens, torch.tensor(parents, dtype=I, device=self.dev),
                                                      self.counts, *self.caches)
        self.tables, self.lens = torch.cat([self.tables, t]), torch.cat([self.lens, l])
        self.history += [list(self.history[p]) for p in parents]
        rows, lens = self.pool.fork(self.host_tables, self.host_lens, parents)
        self.host_tables, self.host_lens = self.host_tables + rows, self.host_lens + lens
        self._same_pool()

    def keep(self, rows):
        gone = [b for b in range(len(self.host_lens)) if b not in rows]
        self.counts = self.paged.free_sequences(self.tables, self.lens, torch.tensor(gone, dtype=I, device=self.dev),
                                                self.counts, BLOCK)
        self.pool.free(self.host_tables, self.host_lens, gone)
        at = torch.tensor(rows, dtype=torch.long, device=self.dev)
        self.tables, self.lens = self.tables[at], self.lens[at]
        self.host_tables, self.host_lens = [self.host_tables[b] for b in rows], [self.host_lens[b] for b in rows]
        self.history = [self.history[b] for b in rows]
        self._same_pool()

    def pack(self):
        self.tables, self.counts, used = self.paged.compact_pages(self.tables, self.lens, self.counts, *self.caches)
        self.host_tables, host_used = self.pool.compact(self.host_tables, self.host_lens)
        assert used.item() == host_used and (self.counts[host_used:] == 0).all()
        self._same_pool()

    def tokens(self, new):
        """`new[b]` more tokens of every sequence, through both layers."""
        before = self.lens
        wanted = before + torch.tensor(new, dtype=I, device=self.dev)
        self.tables, self.lens, self.counts = self.paged.extend_sequences(self.tables, before, wanted, self.counts, BLOCK)
        self.host_tables, self.host_lens = self.pool.extend(self.host_tables, self.host_lens, wanted.tolist())
        self._same_pool()
        assert torch.equal(self.lens, wanted)
        total = sum(new)
        seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).to(self.dev)
        starts = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=I, device=self.dev)
        pos = before[seq] + torch.arange(total, dtype=I, device=self.dev) - starts[seq]
        slots = self.tables[seq, (pos // BLOCK).long()] * BLOCK + pos % BLOCK
        outs = []
        for layer in range(LAYERS):
            qkv = torch.randn(total, (HQ + 2 * HK) * D, generator=self.gen).half()
            q, k, v = (x.reshape(total, -1, D) for x in qkv.split([HQ * D, HK * D, HK * D], dim=1))
            on_dev = qkv.to(self.dev)
            view = lambda a, n: on_dev[:, a * D:(a + n) * D].unflatten(1, (n, D))  # noqa: E731
            gq, gk = self.rotary.rotary_embedding(view(0, HQ), view(HQ, HK), pos, self.cos, self.sin, interleaved=True)
            for got, x in ((gq, q), (gk, k)):
                want = S.rotary_embedding_ref(x, pos.cpu(), self.cos.cpu(), self.sin.cpu(), True)
                # fp32 products of entries up to 1.14, and the rounding to fp16
                assert ((got.cpu().double() - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -25 + 8 * 2.0 ** -22).all()
            kc, vc = self.caches[0][layer], self.caches[1][layer]
            self.ops.reshape_and_cache(gk, view(HQ + HK, HK).contiguous(), kc, vc, slots)
            out = self.paged.paged_attention_chunk(gq, kc, vc, self.tables, self.lens, starts)
            if new == [1] * len(new):
                single = self.ops.paged_attention(gq, kc, vc, self.tables.clamp(min=0), self.lens)
                # both within a rounding of the weights and one of the result
                torch.testing.assert_close(single.float(), out.float(), rtol=2.0 ** -9, atol=2.0 ** -9)
            for b, n in enumerate(new):
                at = slice(int(starts[b]), int(starts[b]) + n)
                hk, hv = (torch.cat([h, x.cpu()[at]]) for h, x in zip(self.history[b][layer], (gk, v)))
                self.history[b][layer] = (hk, hv)
                want = _attend(gq[at].cpu(), hk, hv)
                err = (out[at].cpu().double() - want).abs()
                assert (err <= _tolerance(want, gq[at].cpu(), hk, hv)).all(), (b, layer, float(err.max()))
            outs.append((gq, starts, out))
        return outs

    def again(self, outs):
        """The same queries over the caches as they are now."""
        for layer, (gq, starts, out) in enumerate(outs):
            got = self.paged.paged_attention_chunk(gq, self.caches[0][layer], self.caches[1][layer], self.tables, self.lens, starts)
            assert torch.equal(got, out)


def test_a_run_from_prompts_to_beams(dev):
    s = Server(dev)
    s.add(3)
    s.tokens([37, 5, 100])    # prompts, the last one in two chunks
    s.tokens([1, 1, 30])
    s.fork([2, 2, 0, 2])      # beams next to their parents
    for _ in range(18):       # decoding, over the ends of pages
        s.tokens([1] * 7)
    s.keep([1, 3, 4, 5])      # parents and a beam end
    outs = s.tokens([4, 4, 4, 4])  # drafted tokens
    s.pack()
    s.again(outs)             # moved pages, the same results bit for bit
    s.add(1)
    s.tokens([1, 2, 1, 1, 60])  # a prompt among decoding sequences
    s.fork([4, 4])
    s.tokens([1] * 7)
    s.keep([])
    assert (s.counts == 0).all()


def test_a_pool_that_runs_out(dev):
    """Sequences that get no page keep their lengths, and what they hold stays right."""
    s = Server(dev)
    s.add(5)
    s.tokens([300, 300, 300, 300, 290])  # 95 of 96 pages
    tables, granted, counts = s.paged.extend_sequences(s.tables, s.lens, s.lens + 20, s.counts, BLOCK)
    rows, lens = s.pool.extend(s.host_tables, s.host_lens, [n + 20 for n in s.host_lens])
    assert granted.tolist() == lens == [320, 300, 300, 300, 290] and tables.tolist() == rows
    assert counts.tolist() == s.pool.counts
    s.tables, s.lens, s.counts = tables, granted, counts
    children, child_lens, after = s.paged.fork_sequences(tables, granted, torch.tensor([1, 0, 4], dtype=I, device=dev), counts, *s.caches)
    assert child_lens.tolist() == [0, 320, 0] and torch.equal(children[1], tables[0])
    assert after.tolist() == [n + (1 if p in rows[0] else 0) for p, n in enumerate(counts.tolist())]
