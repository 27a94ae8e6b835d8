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


def kernels(name):
    """The text of each kernel of a source that holds TMEM, by its name."""
    found = {}
    for part in re.split(r"__global__", text_of(name))[1:]:
        if "tcgen05.dealloc" in part:
            found[re.search(r"(\w+)\(const __grid_constant__", part).group(1)] = part
    return found


@pytest.mark.parametrize("name,kernel,rings", [
    ("paged_decode.cu", "paged_decode_kernel", {"K_FULL", "V_FULL", "S_FULL", "P_EMPTY"}),
    ("paged_weights.cu", "few_kernel", {"FULL", "S_FULL"}),
    ("paged_weights.cu", "many_kernel", {"RAW_FULL", "Q_FULL", "S_FULL"}),
])
def test_a_block_ends_behind_what_it_has_under_way(name, kernel, rings):
    """A wait that runs out (which cannot be provoked here) lets warps leave their loops with copies into shared memory or MMAs into TMEM on their way: the warp that
    began them waits for each ring's last ones ahead of the block's last barrier."""
    text = kernels(name)[kernel]
    last = text.rindex("__syncthreads")
    assert set(re.findall(r"last_phases\(bar\(L::(\w+)\)", text[:last])) == rings
    # nothing else is begun: copies come through bring_unit (a ring each) or tma_load_3d, products through umma_commit
    assert len(re.findall(r"bring_unit<", text)) + len(re.findall(r"tma_load_3d\(", text)) == len(rings & {"K_FULL", "V_FULL", "FULL", "RAW_FULL", "Q_FULL"})


def test_every_kernel_with_tensor_memory_is_looked_at():
    assert {k for p in CSRC.glob("paged_*.cu") for k in kernels(p.name)} == {"paged_decode_kernel", "few_kernel", "many_kernel"}


@pytest.mark.parametrize("name,kernel", [("paged_decode.cu", "paged_decode_kernel"), ("paged_weights.cu", "few_kernel"), ("paged_weights.cu", "many_kernel")])
def test_loops_are_left_by_whole_warps(name, kernel):
    """A wait that runs out for single lanes only marks them; what leaves a loop is the vote of a warp, or a comparison that is the same in all its lanes."""
    body = kernels(name)[kernel]
    body = body[:body.rindex("tcgen05.dealloc")]
    for line in body.splitlines():
        if re.search(r"\bmbar_wait(_both_lane)?\(", line):
            assert re.search(r"failed = true;", line), line.strip()
        for left in re.findall(r"(.*)\b(?:break|return false);", line):
            assert re.search(r"!ok\b|!wait_warp\(|!mbar_wait_both\(|!free\(\)|row >= rows", left), line.strip()
