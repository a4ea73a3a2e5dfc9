"""The products' kernels keep what threads store and load by themselves out of the bytes that bulk-tensor copies fill: ordinary accesses and copies go to shared
memory by ways that a barrier alone does not order, and a copy was seen to overtake ordinary reads. Checked on the sources: every pointer into shared memory begins
behind the stages, which are the copies' targets."""
import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "c0ven_b200" / "csrc"


def text_of(path):
    return re.sub(r"//[^\n]*", "", path.read_text())


def behind_the_stages(text):
    """Names of the offsets into shared memory that lie behind the stages: what begins where they end, and what is added to such an offset."""
    made = dict(re.findall(r"static constexpr uint32_t (k\w+) = ([^;]*);", text))
    found = {name for name, of in made.items() if of == "kStages * kStageBytes"}
    while True:
        more = {name for name, of in made.items() if of.split(" + ")[0] in found} - found
        if not more:
            return found
        found |= more


def pointers(text):
    """(pointer, what it begins at) for every one that is made from the kernel's shared memory by a cast."""
    return re.findall(r"(\w+) = \((?:volatile )?\w+ \*\)\(?smem\b\s*(?:\+ (?:SM::)?(\w+))?", text)


@pytest.mark.parametrize("name", ["i8_experts.cu", "mx4_experts.cu"])
def test_no_pointer_into_the_stages(name):
    text = text_of(CSRC / name)
    assert "smem + s * SM::kStageBytes" in text  # the copies' targets
    behind, made = behind_the_stages(text), pointers(text)
    assert {p for p, _ in made} >= {"bars", "first_row", "tile_expert", "warp_part"}
    assert not [p for p in made if p[1] not in behind], made


def test_the_check_sees_a_pointer_into_the_stages():
    text = "static constexpr uint32_t kScales = kStages * kStageBytes;\nstatic constexpr uint32_t kBars = kScales + 4 * N;\nstatic constexpr uint32_t kStageBytes = 128 + 1;"
    assert behind_the_stages(text) == {"kScales", "kBars"}
    assert pointers("uint32_t *a = (uint32_t *)smem;  uint64_t *b = (uint64_t *)(smem + SM::kBars);") == [("a", ""), ("b", "kBars")]
