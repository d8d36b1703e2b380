"""Attention over 4-bit pages within the narrow bounds of int4_exact.py, at the borders of tiles, blocks and splits, through each
kernel: every key counts, and so does every block's scale."""
import pytest

import int4_exact
from test_gpu_int4_pages import run_attn
from test_gpu_paged_edges import HEADS, through

pytestmark = pytest.mark.gpu

PATHS = ["stream", "tiles", "image"]


@pytest.mark.parametrize("d,heads,kv", [*HEADS, (128, 7, 1), (64, 4, 1)])
@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("shape", range(len(int4_exact.SHAPES)))
def test_every_key_counts(gpu_lib, shape, path, d, heads, kv):
    """For the bounds that the call knows and for a max_ctx that leaves the last split all keys but the first 64."""
    new, ctx = int4_exact.SHAPES[shape]
    c = through(path, shape, new, ctx, heads, kv, d, of=int4_exact.batch, page=[16, 64, 32][shape % 3])
    for own in (True, False):
        int4_exact.check(c, *run_attn(c, own=own), path == "stream", own)
    if path != "image":
        int4_exact.check(c, *run_attn(c, max_ctx=64), path == "stream")


@pytest.mark.parametrize("d,heads,kv", HEADS)
@pytest.mark.parametrize("path", PATHS)
def test_every_key_counts_in_option_rows(gpu_lib, path, d, heads, kv):
    c = through(path, 67, [24, 40, 1], [63, 65, 128], heads, kv, d, of=int4_exact.batch, rows=8, page=32)
    int4_exact.check(c, *run_attn(c), path == "stream")


@pytest.mark.parametrize("d,heads,kv", [*HEADS, (128, 32, 1)])
def test_every_key_counts_of_long_states(gpu_lib, d, heads, kv):
    """One and several splits of some thousand keys, tokens of one column of 16 slots and of two."""
    for new, ctx in (([1, 1, 1], [3001, 64, 1500]), ([9], [2049])):
        c = through("stream", 68, new, ctx, heads, kv, d, of=int4_exact.batch, page=64)
        int4_exact.check(c, *run_attn(c, max_new=max(new), max_ctx=max(ctx)), True)
