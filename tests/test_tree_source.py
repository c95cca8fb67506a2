"""What no run of the tree attention can show: rules of its source that keep a wait that
gives up from hanging the GPU and a copy from racing with ordinary accesses."""
from __future__ import annotations

import re
from pathlib import Path

SOURCE = Path(__file__).resolve().parent.parent / "deepseekrpc_b200" / "csrc" / "tree_mla.cu"


def code():
    return re.sub(r"//[^\n]*", "", SOURCE.read_text())


def test_the_schedules_scratch_is_no_place_that_tma_writes():
    """A CTA barrier orders ordinary accesses among themselves, not against the copies that
    TMA writes into the ring, the rotary block or the query afterwards."""
    text = code()
    first = re.search(r"warp_units\s*=\s*reinterpret_cast<int64_t\*>\(([^)]*)\)", text)
    assert first and first.group(1).strip() == "smem + L::kScratchOff"
    assert re.search(r"static_assert\(kScratchOff >= kQOff \+ 9 \* N \* 128", text)
    # every generic pointer into the block names a place of its own
    assert not re.search(r"reinterpret_cast<[^>]*\*>\(smem\)", text)


def test_a_warp_has_one_answer_to_a_wait():
    """A wait that gives up may answer one lane otherwise than another; an aligned
    instruction behind it would then run in a part of the warp.  Outside the helper that
    asks all lanes, only the copying lane, alone in its branch, waits by itself."""
    text = code()
    helper = re.search(r"bool tree_wait_warp\([^{]*\{(.*?)\n\}", text, re.S)
    assert helper and "__all_sync(~0u, tree_wait(" in helper.group(1)
    alone = re.search(r"for \([^;]*; lane == 0 && .*?\n      \}\n", text, re.S)
    assert alone and alone.group(0).count("tree_wait(") == 2
    rest = text.replace(helper.group(0), "").replace(alone.group(0), "")
    assert len(re.findall(r"\btree_wait\(", rest)) == 1  # its definition
