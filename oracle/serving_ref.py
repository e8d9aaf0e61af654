"""Plain definitions, in 64 bits and one sequence, page or pair at a time, of the operators that serve from the paged
caches beyond the reference's surface: attention of a chunk of new tokens, rotary positions, pages.  CPU tensors only;
tests and ``smoke()`` compare the GPU results with these."""
from __future__ import annotations

import math

import torch

from oracle.ops_ref import gather_kv_from_cache


def paged_attention_chunk_ref(q, key_cache, value_cache, block_tables, context_lens, query_starts, scale=None, window=0):
    """``(o [T, Hq, D], lse [T, Hq])`` in fp64.  Sequence b has the rows ``query_starts[b] .. query_starts[b+1]`` of q,
    which are the last tokens of its context; a row sees the keys up to its own position, ``window`` of them at most.
    A row that sees nothing has output 0 and log-sum-exp -inf; rows of no sequence are NaN in both."""
    rows, hq, d = q.shape
    hkv = key_cache.shape[1] * 16 // d
    block = key_cache.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    o = torch.full((rows, hq, d), math.nan, dtype=torch.float64)
    lse = torch.full((rows, hq), math.nan, dtype=torch.float64)
    for b in range(block_tables.shape[0]):
        begin, end = int(query_starts[b]), int(query_starts[b + 1])
        length = max(0, min(int(context_lens[b]), block_tables.shape[1] * block))
        table = block_tables[b].clamp(0, key_cache.shape[0] - 1)
        k = gather_kv_from_cache(key_cache, table, length, hkv).double()
        v = gather_kv_from_cache(value_cache, table, length, hkv).double()
        for i in range(begin, end):
            at = int(context_lens[b]) - (end - begin) + (i - begin)
            last = min(at + 1, length)
            first = max(0, at - window + 1) if window else 0
            for h in range(hq):
                g = h // (hq // hkv)
                if first >= last:
                    o[i, h], lse[i, h] = 0.0, -math.inf
                    continue
                s = k[first:last, g] @ q[i, h].double() * scale
                m = s.max()
                p = torch.exp(s - m)
                o[i, h] = p @ v[first:last, g] / p.sum()
                lse[i, h] = m + math.log(p.sum())
    return o, lse


def rotary_frequencies_ref(rotary_dim, base, max_position, scaling="none", factor=1.0, original=0, low=1.0, high=4.0,
                           beta_fast=32.0, beta_slow=1.0, pair_factors=None):
    """The angle per position of every pair, and the factor on the table's entries, in Python floats."""
    r, amp, out = rotary_dim, 1.0, []
    if scaling == "ntk":
        base = base * factor ** (r / (r - 2))
    if scaling == "dynamic" and max_position > original:
        base = base * (factor * max_position / original - (factor - 1)) ** (r / (r - 2))
    for j in range(r // 2):
        f = base ** (-2.0 * j / r)
        if scaling == "linear":
            f = f / factor
        elif scaling == "yarn":
            lo = max(math.floor(r * math.log(original / (beta_fast * 2 * math.pi)) / (2 * math.log(base))), 0)
            hi = min(math.ceil(r * math.log(original / (beta_slow * 2 * math.pi)) / (2 * math.log(base))), r - 1)
            ramp = min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f / factor * ramp + f * (1 - ramp)
        elif scaling == "wavelength":
            wave = 2 * math.pi / f
            if wave > original / low:
                f = f / factor
            elif wave >= original / high:
                smooth = (original / wave - low) / (high - low)
                f = (1 - smooth) * f / factor + smooth * f
        elif scaling == "pairs":
            f = f / float(pair_factors[j])
        out.append(f)
    if scaling == "yarn" and factor > 1:
        amp = 0.1 * math.log(factor) + 1
    if scaling == "pairs" and factor > 1:
        amp = math.sqrt(1 + math.log(factor) / math.log(original))
    return out, amp


def rotary_tables_ref(max_position, frequencies, amplitude):
    angle = torch.arange(max_position, dtype=torch.float64)[:, None] * torch.tensor(frequencies, dtype=torch.float64)
    return torch.cos(angle) * amplitude, torch.sin(angle) * amplitude


def rotary_embedding_ref(x, position_ids, cos, sin, interleaved):
    """x [tokens, heads, D]; fp64 result for the table's entries as they are."""
    half = cos.shape[1]
    rows = position_ids.long().clamp(0, cos.shape[0] - 1)
    out = x.double().clone()
    for j in range(half):
        a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        c, s = cos[rows, j].double()[:, None], sin[rows, j].double()[:, None]
        out[:, :, a] = x[:, :, a].double() * c - x[:, :, b].double() * s
        out[:, :, b] = x[:, :, b].double() * c + x[:, :, a].double() * s
    return out


class PoolRef:
    """The page operators on Python lists.  ``moves`` collects ``(source page, destination page, tokens)``."""

    def __init__(self, counts, block):
        self.counts = [max(0, int(c)) for c in counts]
        self.block = block
        self.moves = []

    def _tokens(self, tables, lens, b):
        if not 0 <= b < len(tables):
            return 0
        return max(0, min(lens[b], len(tables[b]) * self.block))

    def _inside(self, page):
        return 0 <= page < len(self.counts)

    def _free(self):
        return [p for p, n in enumerate(self.counts) if n == 0]

    def fork(self, tables, lens, parents):
        width = len(tables[0]) if tables else 0
        free, rows, out = self._free(), [], []
        for parent in parents:
            full, part = divmod(self._tokens(tables, lens, parent), self.block)
            if part and not free or full + part == 0:
                rows.append([-1] * width)
                out.append(0)
                continue
            row = tables[parent][:full]
            for page in row:
                if self._inside(page):
                    self.counts[page] += 1
            if part:
                page = free.pop(0)
                self.counts[page] += 1
                if self._inside(tables[parent][full]):
                    self.moves.append((tables[parent][full], page, part))
                row = row + [page]
            rows.append(row + [-1] * (width - len(row)))
            out.append(full * self.block + part)
        return rows, out

    def extend(self, tables, lens, wanted):
        free, rows, out, asked = self._free(), [], [], 0
        for b, want in enumerate(wanted):
            have = self._tokens(tables, lens, b)
            row = list(tables[b])
            if want > have and want <= len(row) * self.block:
                first, need = -(-have // self.block), -(-want // self.block) - -(-have // self.block)
                if need == 0 or asked + need <= len(free):
                    for k in range(need):
                        row[first + k] = free[asked + k]
                        self.counts[free[asked + k]] += 1
                    have = want
                asked += need
            rows.append(row)
            out.append(have)
        return rows, out

    def free(self, tables, lens, which):
        for b in which:
            for j in range(-(-self._tokens(tables, lens, b) // self.block)):
                if self._inside(tables[b][j]):
                    self.counts[tables[b][j]] = max(0, self.counts[tables[b][j]] - 1)

    def compact(self, tables, lens):
        used = sum(n > 0 for n in self.counts)
        holes = [p for p in range(used) if self.counts[p] == 0]
        movers = [p for p in range(used, len(self.counts)) if self.counts[p] > 0]
        to = dict(zip(movers, holes))
        for src, dst in to.items():
            self.counts[dst], self.counts[src] = self.counts[src], 0
            self.moves.append((src, dst, self.block))
        rows = []
        for b, row in enumerate(tables):
            live = -(-self._tokens(tables, lens, b) // self.block)
            rows.append([to.get(p, p) if j < live else p for j, p in enumerate(row)])
        return rows, used

    def moved(self, cache):
        """The cache after the collected moves."""
        out = cache.clone()
        for src, dst, n in self.moves:
            out[dst, :, :n] = cache[src, :, :n]
        return out
