"""The library's scratch buffers have one client each: an entry point, or those that the
headers say must not overlap.  Read from the sources, on the CPU."""
from __future__ import annotations

import re

from conftest import PKG_DIR

CSRC = PKG_DIR / "csrc"

# files whose entry points the headers name together
TOGETHER = [{"paged_attention.hip", "attention_shared.hip"}, {"logprobs.hip", "beam.hip"},
            {"matvec.hip", "pq2_mx.hip"}]


def test_one_client_a_buffer():
    text = (CSRC / "common.hpp").read_text()
    slots = dict(re.findall(r"constexpr int (kScratch\w+) = (\d+);", text))
    count = int(slots.pop("kScratchSlots"))
    assert sorted(int(n) for n in slots.values()) == list(range(count))
    users = {}
    for path in CSRC.iterdir():
        if path.suffix in (".hip", ".cpp", ".hpp"):
            for call in re.findall(r"device_scratch\(([^;]*);", path.read_text()):
                for name in re.findall(r"kScratch\w+", call):
                    users.setdefault(name, set()).add(path.name)
    assert set(users) == set(slots)
    for name, files in users.items():
        assert len(files) == 1 or files in TOGETHER, (name, files)
