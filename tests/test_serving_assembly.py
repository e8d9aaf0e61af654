"""Checks of the compiler's assembly for the kernels around the paged caches (no GPU): no matrix-core result is read before
it is written, no packed fp32 arithmetic, no scratch in the kernels that move pages and rotate."""
import importlib.util
import os
import re

import pytest

import mfma_hazard_scan as scanner

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHUNK = [f"paged_attention_chunk_d{i}.hip" for i in range(4)]


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
