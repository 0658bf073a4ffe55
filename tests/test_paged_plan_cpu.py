"""The launch that paged_attention makes (tg_paged_attention_plan; without a device that of 256 compute units), and which of
them the tests on the GPU reach."""
import pytest

from tokengate_amd import _lib

# sequences, longest segment, most keys, rows, heads, KV heads
SIZES = [(n, q, k, n * q - (n * q) // 5, H, Hkv) for n in (1, 2, 3, 12, 64, 65, 300) for q in (1, 33, 200, 700, 1100)
         for k in (q, 4099, 40000) for H, Hkv in ((16, 8), (5, 5), (16, 2))]


def test_tiles_of_every_launch():
    """A workgroup finds its tile among a sequence's tiles that are not split, by a division by their number: a launch with
    workgroups of such tiles has some."""
    for s in SIZES:
        for ws in (None, 0):
            waves, groups, chunks, split, tiles, order = _lib.paged_plan(*s, workspace_bytes=ws)
            assert tiles >= 1 and 0 <= split <= tiles and (split < tiles or order == 0), (s, ws)
            assert chunks >= 1 and (ws is None or chunks == 1) and waves % groups == 0, (s, ws)


def test_bad_sizes():
    for s in ((0, 8, 8, 8, 2, 1, 0), (1, 0, 8, 8, 2, 1, 0), (1, 8, -1, 8, 2, 1, 0), (1, 8, 8, 0, 2, 1, 0), (1, 8, 8, 8, 3, 2, 0),
              (1, 8, 8, 8, 2, 1, -1)):
        with pytest.raises(RuntimeError, match="bad sizes"):
            _lib.paged_plan(*s)
