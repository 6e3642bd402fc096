"""The Python extension: what a missing one costs, and when it is rebuilt."""

import subprocess
import sys
from pathlib import Path

from batchstream_inference_engine_b200 import build

ROOT = Path(__file__).resolve().parent.parent

WITHOUT = """
import sys
sys.modules["batchstream_inference_engine_b200._native"] = None  # does not load
import torch
from batchstream_inference_engine_b200 import backend, ops
assert ops.kernel_launches() == 0  # the library is there
assert ops.rope_frequencies(8, 1e4, device="cpu")[0].numel() == 4
try:
    ops.rms_norm(torch.zeros(1, 4), torch.zeros(4), 1e-6)
except RuntimeError as e:
    assert "CUDA tensor" in str(e)  # its own refusal
t = torch.zeros(1, 1, 1, 1, 1)
for call in (lambda: ops.copy_blocks(t, t, t, t),
             lambda: ops.window_attention_batched(t, t, t, t, t, 1.0, 1)):
    try:
        call()
    except ImportError as e:
        assert "batchstream_inference_engine_b200.build" in str(e)
    else:
        raise AssertionError("no error")
"""


def test_operators_without_the_extension_still_work():
    done = subprocess.run([sys.executable, "-c", WITHOUT], cwd=ROOT, capture_output=True,
                          text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


def test_the_extension_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    binding = tmp_path / "_native.so"
    binding.write_text("built")
    monkeypatch.setattr(build, "BINDING", binding)
    monkeypatch.setattr(build, "BINDING_FOR", tmp_path / "native_for.txt")
    commands = []

    def run(cmd, **kw):
        commands.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    build.build_binding()  # nothing says what the old one was built against
    build.build_binding()
    assert len(commands) == 1
    monkeypatch.setattr(build, "version", lambda name: "99.0")
    build.build_binding()
    build.build_binding()
    assert len(commands) == 2
