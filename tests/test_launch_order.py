"""Orders inside the kernels, read from their sources.

Programmatic dependent launch: a kernel lets the next one start (pdl_trigger) only after
its own wait (pdl_wait), so a kernel that reads ahead of its wait can only meet the one
just ahead of it.  Tensor memory and cluster barriers: every .aligned instruction that
diverged lanes may reach has a warp barrier just ahead."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "batchstream_inference_engine_b200" / "csrc"
# Their dependents wait before they read: the prefill behind its plan, and with
# lens_ready the merge pass behind the decode.
WAITING_DEPENDENTS = {"prefill_plan_kernel"}


def kernels():
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        starts = list(re.finditer(r"__global__\s+void[^{;]*?(\w+_kernel)\s*\(", text))
        for i, m in enumerate(starts):
            end = starts[i + 1].start() if i + 1 < len(starts) else len(text)
            yield m.group(1), text[m.end(): end]


def test_kernels_trigger_after_their_wait():
    seen = set()
    for name, body in kernels():
        trigger = body.find("pdl_trigger();")
        if trigger < 0 or name in WAITING_DEPENDENTS:
            continue
        seen.add(name)
        wait = body.find("pdl_wait();")
        assert 0 <= wait < trigger, name
    assert {"copy_blocks_kernel", "rotary_append_kernel", "decode_mma_kernel"} <= seen


def sources():
    for path in [*sorted(CSRC.glob("*.cu")), *sorted(CSRC.glob("*.cuh"))]:
        yield path.name, re.sub(r"//[^\n]*", "", path.read_text())


def test_aligned_instructions_follow_a_warp_barrier():
    found = 0
    for name, text in sources():
        for m in re.finditer(r'asm volatile\(\s*"(tcgen05\.(?:alloc|dealloc)|'
                             r'barrier\.cluster\.arrive)\.', text):
            found += 1
            assert re.search(r"__syncwarp\(\);\s*$", text[: m.start()]), (name, m.group(1))
    assert found == 5


def loops(text):
    """Bodies of the for loops of a source, nested ones on their own too."""
    for m in re.finditer(r"\bfor \([^{;]*;[^{;]*;[^{]*\) \{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield text[m.end(): at - 1]


def test_lanes_meet_between_tensor_memory_loads():
    # A loop that loads rows from tensor memory and stores only those that hold a token,
    # or masks some of their keys, brings its lanes together before the next load.
    found = 0
    for name, text in sources():
        for body in loops(text):
            if "tmem_ld32(" in body and re.search(r"\b(store|live)\b", body):
                found += 1
                assert "__syncwarp();" in body, (name, body[:200])
    assert found == 3
