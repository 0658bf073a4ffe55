"""Shapes of paged_attention calls and the launch that each of them takes: waves of a workgroup, key groups among them, whether
tiles' keys are cut into chunks, whether tiles come by the keys they read."""
from typing import List, NamedTuple


class Form(NamedTuple):
    name: str
    new: List[int]
    used: List[int]
    H: int
    Hkv: int
    waves: int
    groups: int
    split: bool
    by_keys: int


def _ragged(n, q, k):
    """Segments up to q of sequences up to k, uneven; the first is the longest in both."""
    new = [max(1, q - (q * (7 * b % 11)) // 16) for b in range(n)]
    return new, [max(m, k - (k * (5 * b % 13)) // 17) for b, m in enumerate(new)]


FORMS = [
    Form("one, four waves", [5], [40], 16, 8, 4, 1, False, 0),
    Form("one, four waves, a head", [5], [40], 5, 5, 4, 1, False, 0),
    Form("one, four waves, chunks", [16], [2500], 16, 8, 4, 1, True, 0),
    Form("one, four waves, a head, chunks", [5], [2500], 5, 5, 4, 1, True, 0),
    Form("one, two groups", [1500], [3000], 16, 8, 8, 2, False, 0),
    Form("one, two groups, a head", [8192], [9000], 5, 5, 8, 2, False, 0),
    Form("one, two groups, chunks", [33], [32769], 16, 8, 8, 2, True, 0),
    Form("one, two groups, a head, chunks", [200], [20000], 5, 5, 8, 2, True, 0),
    Form("one, four groups", [700], [1000], 16, 8, 8, 4, False, 0),
    Form("one, four groups, a head", [200], [400], 1, 1, 8, 4, False, 0),
    Form("one, four groups, chunks", [17], [5000], 16, 8, 8, 4, True, 0),
    Form("one, four groups, a head, chunks", [17], [5000], 5, 5, 8, 4, True, 0),
    Form("one, eight waves, chunks", [100], [32769], 16, 8, 8, 1, True, 0),
    Form("one, eight waves, a head, chunks", [1500], [32769], 1, 1, 8, 1, True, 0),
    Form("many, eight waves", *_ragged(70, 150, 300), 16, 8, 8, 1, False, 0),
    Form("many, eight waves, a head", *_ragged(70, 300, 350), 4, 4, 8, 1, False, 0),
    Form("long, eight waves", *_ragged(9, 1030, 4200), 16, 8, 8, 1, False, 0),
    Form("long, chunks", [1100, 1030], [40000, 38001], 8, 4, 4, 1, True, 0),
    Form("many, chunks, a head", *_ragged(66, 9, 2000), 3, 3, 4, 1, True, 0),
    Form("by keys, four waves", *_ragged(30, 5, 55), 8, 4, 4, 1, False, 1),
    Form("by keys, four waves, a head", *_ragged(8, 16, 16), 5, 5, 4, 1, False, 1),
    Form("by keys, chunks", *_ragged(8, 200, 6000), 16, 8, 4, 1, True, 1),
    Form("by keys, chunks, a head", *_ragged(4, 100, 5000), 5, 5, 4, 1, True, 1),
    Form("by keys, eight waves", *_ragged(20, 150, 160), 16, 8, 8, 1, False, 1),
    Form("by keys, eight waves, a head", *_ragged(40, 200, 300), 5, 5, 8, 1, False, 1),
    Form("by keys, two groups", *_ragged(12, 130, 300), 8, 4, 8, 2, False, 1),
    Form("by keys, two groups, a head", *_ragged(3, 100, 1000), 5, 5, 8, 2, False, 1),
]
