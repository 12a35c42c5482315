"""Every kernel whose shared-memory limit is raised once per device has a slot of its own: with a shared one, whichever kernel
came second kept the default limit, and its launch failed."""
from __future__ import annotations

import re

from min_fa3_demo_b200 import build


def test_slots_are_not_shared():
    slots = {}
    for path in sorted(build.CSRC_DIR.glob("*.cu*")):
        for slot in re.findall(r"once_per_device\([\w.]+,\s*(\d+)\s*,", path.read_text()):
            slots.setdefault(int(slot), []).append(path.name)
    assert slots and all(len(names) == 1 for names in slots.values()), slots
    limit = int(re.search(r"slot >= (\d+)", (build.CSRC_DIR / "b2a_host.cu").read_text()).group(1))
    assert max(slots) < limit
