"""What can be read off the sources of the paged kernels and not be provoked on a device."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "miinfer_b200" / "csrc"


def text_of(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


@pytest.mark.parametrize("name", sorted(p.name for p in CSRC.glob("paged_*.cu")))
def test_sums_of_many_threads_are_of_whole_numbers(name):
    """A sum that threads add to in the order in which they come is one number only where the order does not matter."""
    text = text_of(name)
    for target in re.findall(r"atomicAdd\(&(?:\w+\.)?(\w+)", text):
        kinds = re.findall(r"\b(float|double|uint32_t|int|unsigned long long|uint64_t)\*?\s(?:[\w\[\]]+,\s)*" + target + r"\b", text)
        assert kinds and not {"float", "double"} & set(kinds), (target, kinds)
