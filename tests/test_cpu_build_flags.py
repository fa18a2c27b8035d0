"""Every line that compiles device code turns the packed float32 instructions off (some of their forms are not dependable on this hardware)."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_device_code_is_compiled_without_packed_float32_instructions():
    found = 0
    for folder in ("nvblox_mindmap_amd", "tools", "benchlib", "oracle"):
        for path, _, names in os.walk(os.path.join(ROOT, folder)):
            for name in names:
                if not re.search(r"(\.(py|sh|hip|h|md|txt)|^Makefile)$", name):
                    continue
                with open(os.path.join(path, name), encoding="utf-8", errors="replace") as f:
                    for line in f:
                        if re.search(r"--offload-arch=\S+ -O\d", line):
                            assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, (name, line)
                            found += 1
    assert found >= 4
