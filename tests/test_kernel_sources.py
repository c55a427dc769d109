"""Rules of the kernels that keep a GPU from hanging, read off their sources. A violation could not be
shown by running it: it would hang."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

from qtts_b200.build import SRC_DIR


def kernels(path: Path) -> dict[str, str]:
    """Name -> text from `__global__` to the next one (or the file's end), comments taken out."""
    text = re.sub(r"//[^\n]*", "", path.read_text())
    found = {}
    for part in text.split("__global__")[1:]:
        name = re.search(r"(\w+)\s*\(\s*(?:const\s|uint|int|void|\w+\s)", part[part.index("void") + 4:])
        found[name.group(1)] = part
    return found


WITH_TENSOR_MEMORY = [(p, n, t) for p in sorted(SRC_DIR.glob("*.cu")) for n, t in kernels(p).items() if "tmem_alloc(" in t]


def test_kernels_with_tensor_memory_are_found():
    assert {n for _, n, _ in WITH_TENSOR_MEMORY} >= {"kv4_prompt_kernel", "umma_w8a16_kernel"}


@pytest.mark.parametrize("path,name,text", WITH_TENSOR_MEMORY, ids=[n for _, n, _ in WITH_TENSOR_MEMORY])
def test_dependents_are_released_once_tensor_memory_is_held(path, name, text):
    # A dependent kernel that took columns first would wait (griddepcontrol.wait) for this grid while
    # this grid waits for those columns.
    alloc = text.index("tmem_alloc(")
    published = text.index("__syncthreads()", alloc)
    released = [m.start() for m in re.finditer(r"pdl_launch_dependents\(\)", text)]
    assert released and min(released) > published, f"{path.name}: {name}"


def test_a_wait_that_runs_out_is_the_whole_warps():
    # The prompt kernel's roles go on with warp-wide reductions, ballots and tensor-memory accesses after
    # a wait: lanes that gave up one by one would leave the others of their warp waiting without a limit.
    text = kernels(SRC_DIR / "kv4_prompt.cu")["kv4_prompt_kernel"]
    waits = [m.start() for m in re.finditer(r"mbar_wait_bounded\(", text)]
    assert waits
    for at in waits:
        assert re.search(r"__all_sync\(\s*0xffffffffu,\s*$", text[:at]), text[max(0, at - 90):at + 60]
