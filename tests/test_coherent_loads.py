"""Loads of kernels that are launched before the kernel just ahead of them has ended, read from
their sources."""

import re

from .test_launch_order import sources

# Pointers of kernels that are launched early to what the framework's kernel just ahead of
# them may write: lengths and rows (step metadata, lists of chunks), pools (appends), logits.
WRITTEN_AHEAD = r"context_lens|seq_rows|cu_q|chunk_rows|codes|scales|bytes|logits|\bp\)"
EARLY = ("decode.cuh", "decode_join.cuh", "decode_int4.cu", "decode_mma.cu", "window.cuh",
         "window_prefill.cu", "window_simt.cu", "drafts.cu", "int4_cache.cu")


def test_kernels_launched_early_read_what_is_written_ahead_coherently():
    # (The read-only path does not wait for the kernel ahead: tables alone go by it, which
    # no kernel writes.)
    seen = set()
    for name, text in sources():
        if name not in EARLY:
            continue
        seen.add(name)
        for m in re.finditer(r"__ldg\(((?:[^()]|\([^()]*\)|\((?:[^()]|\([^()]*\))*\))*)\)", text):
            assert not re.search(WRITTEN_AHEAD, m.group(1) + ")"), (name, m.group(0))
            assert "table" in m.group(1), (name, m.group(0))
    assert seen == set(EARLY)


def test_coherent_loads_stay_behind_the_wait():
    text = dict(sources())["common.cuh"]
    loads = re.findall(r"coherent_load\([^)]*\) \{(.*?)\n\}", text, re.S)
    assert len(loads) >= 4
    for body in loads:
        assert re.search(r'asm volatile\(\s*"ld\.global\.', body) and ".nc" not in body
