"""Programmatic dependent launch, read from the kernels' sources: a kernel lets the next
one start (pdl_trigger) only after its own wait (pdl_wait), so a kernel that reads
ahead of its wait can only meet the one just ahead of it."""

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
