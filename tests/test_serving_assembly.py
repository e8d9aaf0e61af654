"""Checks of the compiler's assembly for the kernels around the paged caches (no GPU): no matrix-core result is read before
it is written, no packed fp32 arithmetic, no scratch in the kernels that move pages and rotate."""
import importlib.util
import os
import re

import pytest

import mfma_hazard_scan as scanner

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHUNK = [f"paged_attention_chunk_d{i}.hip" for i in range(8)]


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    spec = importlib.util.spec_from_file_location("aops_build", os.path.join(ROOT, "ascend-ops_amd", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    names = CHUNK + ["paged_attention_chunk.hip", "pages.hip", "rotary.hip"]
    return {n: p.read_text() for n, p in zip(names, build.emit_assembly(tmp_path_factory.mktemp("asm"), names))}


def test_no_matrix_core_result_is_read_early(assembly):
    seen = 0
    for name in CHUNK:
        found = scanner.scan(assembly[name])
        assert not found, f"{name}: {found[:5]}"
        seen += assembly[name].count("v_mfma_")
    assert seen > 1000


def test_no_packed_fp32_and_no_generic_addresses(assembly):
    for name, text in assembly.items():
        assert not re.search(r"v_pk_(?:add|mul|fma)_f32", text), name
        assert not re.search(r"\bflat_(?:load|store)", text), name


def test_no_scratch(assembly):
    for name in ("pages.hip", "rotary.hip", "paged_attention_chunk.hip"):
        sizes = re.findall(r"amdhsa_private_segment_fixed_size (\d+)", assembly[name])
        assert sizes and set(sizes) == {"0"}, name


def _chunk_kernels(text):
    """(kind, head size, body lines) of every chunk attention kernel."""
    for m in re.finditer(r"^(_ZN4aops\d+chunk_(tiles|shares)_kernelILi(\d+)E\w+):[^\n]*\n(.*?)^\.Lfunc_end", text, re.S | re.M):
        lines = (line.split(";")[0].strip() for line in m.group(4).split("\n"))
        yield m.group(2), int(m.group(3)), [line for line in lines if line]


def _copies_per_step(d):
    """Fewest copies of a wave per tile of keys, the steps that may be on their way behind a counted wait, and whether all
    waves copy the same number."""
    tile, waves = (64 if d <= 176 else 32), (8 if d <= 128 else 4)
    stages = 4 if 16 * tile * d <= 128 * 1024 else 3
    chunks, per_round = d // 16, waves * 64 // (2 * tile)
    return 2 * (chunks // per_round) + 1, stages - 2, chunks % per_round == 0


def test_copies_to_lds_and_their_waits(assembly):
    """The copies are assembly that the compiler does not count.  Each is its three instructions, which alone use M0; a
    wait that leaves some on their way leaves no more than the last steps', and follows its step's copies."""
    kernels = counted = 0
    for name in CHUNK:
        for kind, d, lines in _chunk_kernels(assembly[name]):
            kernels += 1
            where = f"chunk_{kind}_kernel<{d}>"
            m0 = {i for i, line in enumerate(lines) if re.search(r"\bm0\b", line)}
            for i, line in enumerate(lines):
                if line.startswith("global_load_lds"):
                    assert re.match(r"s_mov_b32 m0, s\d+$", lines[i - 2]) and lines[i - 1] == "s_nop 0", where
                    m0.discard(i - 2)
            assert not m0, (where, [lines[i] for i in sorted(m0)][:5])
            copies, steps, all_waves_alike = _copies_per_step(d)
            in_block = 0
            waited = False
            for line in lines:
                if line.endswith(":") or line.startswith(("s_branch", "s_cbranch", "s_endpgm")):
                    in_block, waited = 0, False
                elif line.startswith("global_load_lds"):
                    in_block += 1
                    assert not waited, where  # a copy behind its step's wait would be counted with the next step's
                elif re.match(r"s_waitcnt vmcnt\(\d+\) lgkmcnt\(0\)$", line) and in_block:
                    n = int(re.search(r"vmcnt\((\d+)\)", line).group(1))
                    if n:
                        # (where only some waves copy in a step's last round, that is a branch)
                        assert n == steps * copies and in_block >= (copies if all_waves_alike else 1), (where, n, in_block)
                        counted += 1
                        waited = True
    assert kernels == 32 and counted >= 32, (kernels, counted)


def test_lds_is_written_before_a_barrier(assembly):
    """The barriers of the loops are bare: a wave waits for its own LDS writes in front of them."""
    barriers = 0
    for name in CHUNK:
        for kind, d, lines in _chunk_kernels(assembly[name]):
            pending = None
            for line in lines:
                if line.startswith("ds_write"):
                    pending = line
                elif line.startswith("s_waitcnt") and "lgkmcnt(0)" in line:
                    pending = None
                elif line == "s_barrier":
                    barriers += 1
                    assert pending is None, (f"chunk_{kind}_kernel<{d}>", pending)
    assert barriers > 500


def test_tile_kernels_keep_their_registers(assembly):
    for name in CHUNK:
        sizes = re.findall(r"\.amdhsa_kernel _ZN4aops\d+chunk_tiles_kernel\w+\n.*?private_segment_fixed_size (\d+)", assembly[name], re.S)
        assert len(sizes) == 2 and set(sizes) == {"0"}, name


def _loads_together(lines):
    """Numbers of memory loads that are issued without a wait for one, or a branch, between them."""
    found, run = [], 0
    for line in lines + ["s_branch"]:
        if re.match(r"global_load_(?!lds)", line):
            run += 1
        elif "vmcnt" in line or line.startswith(("s_branch", "s_cbranch")):
            found += [run] if run else []
            run = 0
    return found


def test_counts_of_pages_are_loaded_together(assembly):
    """A lane's eight counts of a pass over the pool are on their way at once, in every kernel that makes such passes."""
    passes = {"compact_plan_kernel": 2, "fork_small_kernel": 3, "extend_small_kernel": 4, "compact_small_kernel": 2, "pages_plan_kernel": 1}
    seen = dict.fromkeys(passes, 0)
    for m in re.finditer(r"^_ZN4aops\d+(\w+?_kernel)\w*:[^\n]*\n(.*?)^\.Lfunc_end", assembly["pages.hip"], re.S | re.M):
        if m.group(1) in passes:
            seen[m.group(1)] += 1
            lines = [line.split(";")[0].strip() for line in m.group(2).split("\n")]
            assert sum(n == 8 for n in _loads_together(lines)) >= passes[m.group(1)], m.group(1)
    assert seen == {**dict.fromkeys(passes, 1), "pages_plan_kernel": 2}, seen


def test_bounds_of_sequences_are_loaded_together(assembly):
    """A lane that looks for a tile among eight sequences has their nine bounds on their way at once."""
    seen = 0
    for name in CHUNK:
        for kind, d, lines in _chunk_kernels(assembly[name]):
            if kind != "tiles":
                continue
            found, dwords = set(), 0
            for line in lines:
                load = re.match(r"global_load_dword(?:x(\d))? ", line)
                if load:
                    dwords += int(load.group(1) or 1)
                elif "vmcnt" in line or line.startswith(("s_branch", "s_cbranch")):
                    found.add(dwords)
                    dwords = 0
            assert 9 in found, (d, found)
            seen += 1
    assert seen == 16
