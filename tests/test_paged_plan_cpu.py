"""The launch that paged_attention makes (tg_paged_attention_plan; without a device that of 256 compute units), and which of
them the tests on the GPU reach."""
import pytest

from paged_forms import FORMS
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
            assert order in (0, 1) and chunks >= 1 and (ws is None or chunks == 1) and waves % groups == 0, (s, ws)


def test_bad_sizes():
    for s in ((0, 8, 8, 8, 2, 1, 0), (1, 0, 8, 8, 2, 1, 0), (1, 8, -1, 8, 2, 1, 0), (1, 8, 8, 0, 2, 1, 0), (1, 8, 8, 8, 3, 2, 0),
              (1, 8, 8, 8, 2, 1, -1)):
        with pytest.raises(RuntimeError, match="bad sizes"):
            _lib.paged_plan(*s)


@pytest.mark.parametrize("form", FORMS, ids=[f.name for f in FORMS])
def test_which_launch_a_shape_takes(form):
    """The kernel that test_paged_forms_gpu.py's shapes are named for."""
    n = len(form.new)
    waves, groups, chunks, _, _, order = _lib.paged_plan(n, max(form.new), max(form.used), sum(form.new) + 2, form.H, form.Hkv)
    assert (waves, groups, chunks > 1, order) == (form.waves, form.groups, form.split, form.by_keys)


def test_every_launch_has_a_shape():
    """Every form that any of many sizes takes, for one query head of a workgroup and for two."""
    def kernel(H, Hkv, plan):
        return plan[0], plan[1], plan[2] > 1, plan[5], 1 + ((H // Hkv) % 2 == 0)
    taken = set()
    for n in (1, 2, 5, 12, 20, 40, 64, 65, 100):
        for q in (1, 16, 33, 100, 130, 200, 700, 1030, 1500, 2320, 8192):
            for k in (q, 2 * q, 1000, 4100, 9000, 20000, 32769, 40000):
                if k >= q:
                    for H, Hkv in ((16, 8), (8, 4), (4, 4), (5, 5), (1, 1), (2, 1)):
                        taken.update(kernel(H, Hkv, _lib.paged_plan(n, q, k, rows, H, Hkv)) for rows in (n * q, q + (n - 1) * q // 2))
    assert taken == {(f.waves, f.groups, f.split, f.by_keys, 1 + ((f.H // f.Hkv) % 2 == 0)) for f in FORMS}
