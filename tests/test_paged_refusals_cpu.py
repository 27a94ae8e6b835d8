"""Arrays of a paged call that lie over one another, scales of other shapes; no GPU needed."""
import pytest
import torch

from miinfer_b200 import kv, paged
from test_paged_cpu import DEVICE, INVALID, attend, batch_of, evict, no_gpu, view_of


@pytest.mark.parametrize("change", [
    dict(new_lengths=12288 + 4), dict(new_lengths=12288 + 8), dict(new_lengths=12288 - 8),                     # the batch's three lengths, in part
    dict(new_lengths=4096 + 4 * 29), dict(new_lengths=8192 + 4 * 3), dict(new_lengths=(1 << 14) - 8),          # its last page, its last start; the target's first page
    dict(kept=12288), dict(kept=4096 - 4 * (3 * 2 * 64 - 1)), dict(kept=8192), dict(kept=(1 << 14) + 4 * 11), dict(new_weights=12288), dict(new_weights=(1 << 14) + 4 * 11),
])
def test_what_an_eviction_writes_lies_over_none_of_the_batch_s_arrays(change):
    assert evict(view_of(), batch_of(), **change) == INVALID


@no_gpu
@pytest.mark.parametrize("change", [dict(new_lengths=12288 + 12), dict(new_lengths=12288 - 12), dict(new_lengths=4096 + 4 * 30), dict(new_lengths=8192 + 4 * 4),
                                    dict(kept=(1 << 14) + 4 * 12), dict(new_weights=12288 - 4 * 3 * 2 * 64), dict(target=4096, pages=10)])
def test_what_an_eviction_writes_may_lie_next_to_them(change):
    assert evict(view_of(), batch_of(), **change) == DEVICE


def test_results_over_queries_that_are_read_again_are_refused():
    """Statistics of fp32 queries over fp16 keys: the queries are read a second time when output and lse are written.  9 rows of 8 heads of 128."""
    v, q, room = view_of(quant_mode=2, key_f16=4096), 1 << 22, 9 * 8 * 128 * 4
    for out, lse in [(q, 1 << 26), (q + room - 16, 1 << 26), (q - room // 2 + 16, 1 << 26), (1 << 24, q), (1 << 24, q + room - 4), (1 << 24, q - 9 * 8 * 4 + 4)]:
        assert attend(v, batch_of(), q=q, q_dtype=1, out=out, lse=lse) == INVALID
    if not torch.cuda.is_available():
        for out, lse in [(q + room, 1 << 26), (q - room // 2, 1 << 26), (1 << 24, q + room), (1 << 24, q - 9 * 8 * 4)]:
            assert attend(v, batch_of(), q=q, q_dtype=1, out=out, lse=lse) == DEVICE


def test_scales_of_other_shapes_are_value_errors():
    q8, q = torch.zeros(4, 2, 16, 128, dtype=torch.int8), kv.KvCacheQuantMode.kQ8Q8
    good = torch.zeros(4, 2, 16, 4, dtype=torch.float16)
    for bad in (torch.zeros(4, 2, 16, dtype=torch.float16), torch.zeros(4, 2, 16, 0, dtype=torch.float16), torch.zeros(4, 2, 16, 4, 1, dtype=torch.float16)):
        for scales in ((bad, good), (good, bad)):
            with pytest.raises(ValueError):
                paged.PagedView.of(q8, scales[0], q8, scales[1], q)
