"""The workspace's parts; no GPU needed."""
from test_paged_cpu import batch_of, size, view_of


def test_a_workspace_has_room_for_mean_keys_where_they_are_used():
    """Statistics of fp32 queries over fp16 keys take a second pass, whose result lies over the copy of V; over int8 keys there is none."""
    v8, v16 = view_of(page_size=256, pages=4000, qblock=128), view_of(page_size=256, pages=4000, qblock=128, quant_mode=2, key_f16=4096)
    b = batch_of(sequences=1, total_tokens=4000, max_tokens=4000, max_length=4000, max_pages=20, total_length=4000)
    assert size(v8, b, 16) < size(v16, b, 16)
